"""tree_attention against the formula in 64 bits, at every edge of nodes, keys, pages and splits.

Up to 16 rows (nodes x heads of a group) to a KV head take one kernel, more another: where that is
not plain from the sizes, tests run with a number of nodes for each.

The bound is :func:`oracle.serving.attention_bound`'s: what rounding scores, probabilities and outputs
to their types allows, for the row's own numbers.
"""
from __future__ import annotations

import math
import random

import pytest
import torch

from oracle import branches
from oracle import serving as ref

gpu = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def _table(lens, page, seed, width=None):
    """A block table over shuffled pages, and the number of pages."""
    rng = random.Random(seed)
    need = [-(-max(n, 0) // page) for n in lens]
    order = list(range(sum(need) + 2))
    rng.shuffle(order)
    table = torch.full((len(lens), width or max(max(need), 1)), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    return table, sum(need) + 2


def _cache(n, kv, page, hd, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(n, kv, page, hd, generator=g).to(dtype).cuda()


def _parents(rng, nodes):
    return [rng.randint(max(-1, j - 5), j - 1) if j else -1 for j in range(nodes)]


def _trees(seqs, nodes, seed):
    from moeinfra_b200 import kernels

    rng = random.Random(seed)
    return torch.stack([kernels.tree_masks(_parents(rng, nodes)) for _ in range(seqs)])


def _bits(visible, nodes):
    """bool [.., nodes, nodes] of a mask."""
    i = torch.arange(nodes)
    return (visible[..., i // 64] >> (i % 64)) & 1 == 1


def _check(q, kp, vp, table, lens, visible, counts=None, scale=None, got=None):
    """Compare with the oracle; q [B, T, H, hd] on the CPU."""
    from moeinfra_b200 import kernels

    B, T, H, hd = q.shape
    at = torch.tensor(lens, dtype=torch.int32, device="cuda")
    n_at = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    if got is None:
        got = kernels.tree_attention(q.cuda(), kp, vp, table.cuda(), at, visible.cuda(), counts=n_at,
                                     scale=scale)
        kernels.check_device()
    sc = hd ** -0.5 if scale is None else scale
    for b, n in enumerate(lens):
        have = T if counts is None else max(counts[b], 0)
        if n < 0 or have == 0:
            assert not got[b].any()
            continue
        assert not got[b, have:].any()
        k, v = (ref.gather_pages(p.cpu(), table[b], n + have).transpose(0, 1) for p in (kp, vp))
        seen = torch.cat((torch.ones(have, n, dtype=torch.bool), _bits(visible[b], T)[:have, :have]), 1)
        want, weight, off = branches.tree_attention(q[b, :have], k, v, seen, sc)
        bound = ref.attention_bound(q.dtype, want, weight, off)
        err = (got[b, :have].double().cpu() - want).abs()
        assert (err <= bound).all(), (b, n, float((err / bound).max()))
    return got


def _q(B, T, H, hd, dtype, seed=3):
    g = torch.Generator().manual_seed(seed + T + H)
    return torch.randn(B, T, H, hd, generator=g).to(dtype)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H,KV,nodes", [(32, 8, 16), (4, 4, 3), (7, 1, 40), (28, 4, 19), (16, 1, 16),
                                        (40, 2, 7), (130, 1, 2), (8, 2, 65), (24, 1, 1)])
def test_heads(dtype, hd, H, KV, nodes):
    """Groups of 1 to 130 heads in one tile, two and several blocks; lengths at steps' and pages' edges."""
    lens = [1, 63, 0, 64, 65, 47, 100]
    table, n = _table([m + nodes for m in lens], 16, 5)
    kp, vp = (_cache(n, KV, 16, hd, dtype, s) for s in (1, 2))
    _check(_q(len(lens), nodes, H, hd, dtype), kp, vp, table, lens, _trees(len(lens), nodes, hd))


@gpu
@pytest.mark.parametrize("lens,page,nodes", [
    ([0], 16, 1), ([1024], 16, 8), ([3000], 64, 5), ([5000, 1, 0, 700], 64, 33),
    ([2047, 2048, 2049], 48, 12), ([257] * 40, 32, 9), ([31, 4000] * 20, 128, 4), ([1] * 300, 16, 2),
    ([-1] * 50 + [1500] + [-1] * 40, 16, 6), ([20000], 16, 70), ([300], 80, 200), ([0, 3], 16, 129),
    ([40000, 7], 96, 3), ([0, 1, 400, 64, -1, 250] * 20, 16, 9), ([0, 1, 700, 64, -1, 250] * 20, 16, 9),
    ([55] * 75, 64, 9), ([119, -1, -1, -1] * 38 + [0], 16, 9)])
def test_lengths(lens, page, nodes):
    """Units in a CTA's share and over many CTAs, several blocks of rows, empty sequences between."""
    H, KV, hd = 8, 2, 64
    table, n = _table([m + nodes if m >= 0 else 0 for m in lens], page, 6)
    kp, vp = (_cache(n, KV, page, hd, torch.float16, s) for s in (3, 4))
    _check(_q(len(lens), nodes, H, hd, torch.float16), kp, vp, table, lens, _trees(len(lens), nodes, 7))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KV", [(32, 8), (32, 1), (64, 1)])
def test_wide_trees_over_cut_units(dtype, H, KV):
    """Two tiles of rows and several blocks, joined over CTAs."""
    lens, nodes, hd = [3001, 64, 517], 64, 128
    table, n = _table([m + nodes for m in lens], 64, 8)
    kp, vp = (_cache(n, KV, 64, hd, dtype, s) for s in (5, 6))
    _check(_q(len(lens), nodes, H, hd, dtype), kp, vp, table, lens, _trees(len(lens), nodes, 9))


@gpu
@pytest.mark.parametrize("KV", [2, 8])
def test_counts_and_rows_without_keys(KV):
    """Trees of different sizes in one call; nodes that see nothing, or only others; no pages needed
    past a tree's own nodes."""
    from moeinfra_b200 import kernels

    lens, counts, nodes = [0, 30, 64, 5, -1, 100], [3, 10, 0, -2, 7, 1], 10
    table, n = _table([max(m, 0) + max(c, 0) for m, c in zip(lens, counts)], 16, 4)
    kp, vp = (_cache(n, KV, 16, 64, torch.float16, s) for s in (7, 8))
    visible = _trees(6, nodes, 3)
    visible[0, 1] = 0                  # sees nothing: no cached positions
    visible[0, 2] = 1 << 9             # sees only a node that is not there
    visible[1, 4] = 0                  # sees the cached positions alone
    visible[1, 5] = -1                 # sees all, later ones too
    q = _q(6, nodes, 8, 64, torch.float16)
    got = _check(q, kp, vp, table, lens, visible, counts)
    assert not got[0, 1].any() and not got[0, 2].any()
    assert got.isfinite().all()
    empty = kernels.tree_attention(q.cuda()[:, :0], kp, vp, table.cuda(),
                                   torch.zeros(6, dtype=torch.int32, device="cuda"),
                                   visible.cuda()[:, :0, :0])
    assert empty.shape == (6, 0, 8, 64)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("lens", [[5, 20], [1500, 64]])
@pytest.mark.parametrize("nodes,KV", [(9, 2), (5, 4)])
def test_what_a_row_does_not_see_has_no_effect(dtype, bad, lens, nodes, KV):
    """Pages past the end, pages of nobody, and nodes outside a row's branch hold NaN or infinities."""
    H, hd, page = 8, 128, 32
    table, n = _table([m + nodes for m in lens], page, 8)
    kp, vp = (_cache(n, KV, page, hd, dtype, s) for s in (5, 6))
    used = {int(p) for row in table for p in row if p >= 0}
    for p in range(n):
        if p not in used:
            kp[p], vp[p] = bad, bad
    for b, m in enumerate(lens):
        if (m + nodes) % page:
            last = int(table[b, (m + nodes) // page])
            kp[last, :, (m + nodes) % page:], vp[last, :, (m + nodes) % page:] = bad, bad
        at = m + 4                     # node 4 is bad: rows that see it are not compared
        kp[int(table[b, at // page]), :, at % page] = bad
        vp[int(table[b, at // page]), :, at % page] = bad
    visible = _trees(2, nodes, 2)
    sees = _bits(visible, nodes)[:, :, 4]
    q = _q(2, nodes, H, hd, dtype)
    from moeinfra_b200 import kernels

    got = kernels.tree_attention(q.cuda(), kp, vp, table.cuda(),
                                 torch.tensor(lens, dtype=torch.int32, device="cuda"), visible.cuda())
    kernels.check_device()
    assert bool(got[sees.cuda()].isnan().any())
    got[sees.cuda()] = 0
    for b, m in enumerate(lens):       # the oracle without node 4's rows
        k, v = (ref.gather_pages(p.cpu(), table[b], m + nodes).transpose(0, 1) for p in (kp, vp))
        seen = torch.cat((torch.ones(nodes, m, dtype=torch.bool), _bits(visible[b], nodes)), 1)
        rows = ~sees[b]
        want, weight, off = branches.tree_attention(q[b, rows], k, v, seen[rows], hd ** -0.5)
        bound = ref.attention_bound(dtype, want, weight, off)
        assert ((got[b].cpu()[rows].double() - want).abs() <= bound).all()


@gpu
@pytest.mark.parametrize("nodes", [3, 10])
def test_scores_of_infinity_and_nan_make_a_row_nan(nodes):
    H, KV, hd, page = 4, 1, 64, 16
    table, n = _table([40 + nodes] * 2, page, 8)
    kp, vp = (_cache(n, KV, page, hd, torch.float16, s) for s in (5, 6))
    q = _q(2, nodes, H, hd, torch.float16).cuda()
    q[0, 1, 2] = math.nan
    q[1, 2, 3] = -math.inf
    from moeinfra_b200 import kernels

    got = kernels.tree_attention(q, kp, vp, table.cuda(), torch.tensor([40, 40], device="cuda").int(),
                                 _trees(2, nodes, 2).cuda())
    kernels.check_device()
    bad = torch.zeros(2, nodes, H, dtype=torch.bool, device="cuda")
    bad[0, 1, 2] = bad[1, 2, 3] = True
    assert bool(got[bad].isnan().all()) and bool(got[~bad].isfinite().all())


@gpu
@pytest.mark.parametrize("nodes", [2, 12])
def test_peaked_and_faint_softmax(nodes):
    """One key far above the others, scores far below zero, and a maximum that keeps growing."""
    H, KV, hd, page, m = 4, 1, 64, 16, 700
    table, n = _table([m + nodes] * 3, page, 2)
    kp = torch.zeros(n, KV, page, hd)
    vp = torch.randn(n, KV, page, hd, generator=torch.Generator().manual_seed(0))
    q = torch.zeros(3, nodes, H, hd)
    q[..., 0] = 1.0
    for b, base in ((0, 0.0), (1, -300.0)):
        kp[table[b, :-(-(m + nodes) // page)].long(), 0, :, 0] = base
        kp[int(table[b, 3]), 0, 5, 0] = base + 11.0
    for j in range(m):
        kp[int(table[2, j // page]), 0, j % page, 0] = j * 0.1
    _check(q.half(), kp.half().cuda(), vp.half().cuda(), table, [m] * 3, _trees(3, nodes, 1), scale=1.0)


@gpu
@pytest.mark.parametrize("nodes", [4, 12])
def test_strided_inputs_shared_pages_and_repeats(nodes):
    """Keys and values side by side, queries from a wider buffer, one mask for all sequences, one page
    in two sequences; the same call twice gives the same bits."""
    from moeinfra_b200 import kernels

    H, KV, hd, page, lens = 8, 2, 128, 16, [40, 2000, 33]
    table, n = _table([m + nodes for m in lens], page, 9)
    table[2, 0] = table[0, 0]
    both = _cache(2 * n, KV, page, hd, torch.bfloat16, 7).view(n, 2, KV, page, hd)
    kp, vp = both[:, 0], both[:, 1]
    wide = torch.randn(3, nodes + 2, 2 * H, hd, generator=torch.Generator().manual_seed(4)).bfloat16()
    q, one = wide.cuda()[:, 1:-1, H:], _trees(1, nodes, 3)
    at = torch.tensor(lens).int().cuda()
    far = torch.full((3, table.shape[1] + 3), -7, dtype=torch.int32, device="cuda")
    far[:, :table.shape[1]] = table.cuda()
    got = kernels.tree_attention(q, kp, vp, far[:, :table.shape[1]], at, one.cuda().expand(3, nodes, 1))
    _check(wide[:, 1:-1, H:].contiguous(), kp.contiguous(), vp.contiguous(), table, lens,
           one.expand(3, nodes, 1), got=got)
    again = kernels.tree_attention(q, kp, vp, table.cuda(), at, one.cuda().repeat(3, 1, 1))
    assert torch.equal(got, again)


@gpu
def test_one_node_is_paged_attention():
    """A single node is the decode step's token, its own position included."""
    from moeinfra_b200 import kernels

    lens = [0, 100, 777]
    table, n = _table([m + 1 for m in lens], 16, 9)
    kp, vp = (_cache(n, 2, 16, 128, torch.float16, s) for s in (1, 2))
    q = _q(3, 1, 8, 128, torch.float16)
    got = _check(q, kp, vp, table, lens, _trees(3, 1, 0))
    want = kernels.paged_attention(q[:, 0].cuda(), kp, vp, table.cuda(),
                                   torch.tensor([m + 1 for m in lens], dtype=torch.int32, device="cuda"))
    # Two results that each round probabilities and outputs: some 2^-10 of a value near 1.
    assert float((got[:, 0].float() - want.float()).abs().max()) < 2.0 ** -8


@gpu
@pytest.mark.parametrize("nodes", [20, 4])
def test_graphs_follow_their_inputs_side_by_side(nodes):
    """Captured calls read lengths, masks and pages at replay; two on one stream, replayed on two."""
    from moeinfra_b200 import kernels

    H, KV, hd, page = 8, 2, 64, 16
    table, n = _table([2500, 2500], page, 3)
    kp, vp = (_cache(n, KV, page, hd, torch.float16, s) for s in (8, 9))
    tab = table.cuda()
    ws = kernels.tree_attention_workspace(kp)
    runs = []
    for i in range(2):
        q = _q(2, nodes, H, hd, torch.float16, i).cuda()
        at, vis = torch.zeros(2, dtype=torch.int32, device="cuda"), _trees(2, nodes, i).cuda()
        kernels.tree_attention(q, kp, vp, tab, at, vis)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = kernels.tree_attention(q, kp, vp, tab, at, vis, workspace=ws if i else None)
        runs.append((g, q, at, vis, out))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn, lens in enumerate(([300, 2100], [0, 17], [2400, -1])):
        for g, q, at, vis, out in runs:
            at.copy_(torch.tensor(lens))
            vis.copy_(_trees(2, nodes, 10 + turn))
        torch.cuda.synchronize()
        for (g, *_), s in zip(runs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for g, q, at, vis, out in runs:
            assert torch.equal(out, kernels.tree_attention(q, kp, vp, tab, at, vis))
    kernels.check_device()


@gpu
@pytest.mark.parametrize("nodes", [3, 20])
def test_bad_lengths_and_pages_are_reported(nodes):
    from moeinfra_b200 import kernels

    H, KV, hd, page = 4, 2, 64, 16
    kp, vp = (_cache(2, KV, page, hd, torch.float16, s) for s in (8, 9))
    q = torch.ones(1, nodes, H, hd, dtype=torch.float16, device="cuda")
    vis = _trees(1, nodes, 0).cuda()
    for table, n, count in (([0, 1], 33 - nodes, nodes), ([0, 7], 32 - nodes, nodes), ([-1, 0], 2, nodes),
                            ([0, 1], 4, nodes + 1), ([0, 1], 2 ** 31 - 1, nodes)):
        kernels.tree_attention(q, kp, vp, torch.tensor([table], dtype=torch.int32, device="cuda"),
                               torch.tensor([n], dtype=torch.int32, device="cuda"), vis,
                               counts=torch.tensor([count], dtype=torch.int32, device="cuda"))
        with pytest.raises(RuntimeError, match="out of range"):
            kernels.check_device()
    kernels.check_device()


@gpu
@pytest.mark.parametrize("nodes", [3, 20])
def test_past_two_to_the_31_elements(nodes):
    """Pages whose elements lie past 2^31 (and bytes past 2^32) of the cache."""
    KV, page, hd = 8, 64, 128
    n = 2 ** 31 // (KV * page * hd) + 40
    kp = torch.zeros(n, KV, page, hd, dtype=torch.float16, device="cuda")
    vp = torch.zeros_like(kp)
    table = torch.tensor([[n - 1, n - 17, 0]], dtype=torch.int32)
    for t, s in ((kp, 1), (vp, 2)):
        t[table[0].long()] = _cache(3, KV, page, hd, torch.float16, s)
    q = _q(1, nodes, 16, hd, torch.float16)
    from moeinfra_b200 import kernels

    got = kernels.tree_attention(q.cuda(), kp, vp, table.cuda(),
                                 torch.tensor([150], dtype=torch.int32, device="cuda"),
                                 _trees(1, nodes, 1).cuda())
    at = table[0].long()
    small = torch.arange(3, dtype=torch.int32)[None]
    _check(q, kp[at], vp[at], small, [150], _trees(1, nodes, 1), got=got)


@gpu
@pytest.mark.parametrize("H,KV,nodes", [(32, 8, 16), (32, 8, 64), (16, 8, 7)])
def test_a_long_batch_many_times(H, KV, nodes):
    """Sequences of some 30 steps each, whose two pipelines drift apart; the same bits every time."""
    from moeinfra_b200 import kernels

    lens, page, hd = [1800 + 7 * i for i in range(48)], 64, 128
    table, n = _table([m + nodes for m in lens], page, 3)
    kp, vp = (_cache(n, KV, page, hd, torch.bfloat16, s) for s in (1, 2))
    q, vis = _q(48, nodes, H, hd, torch.bfloat16), _trees(48, nodes, 3)
    at = torch.tensor(lens, dtype=torch.int32, device="cuda")
    args = (q.cuda(), kp, vp, table.cuda(), at, vis.cuda())
    first = kernels.tree_attention(*args)
    for _ in range(20):
        assert torch.equal(kernels.tree_attention(*args), first)
    kernels.check_device()
    _check(q[45:], kp, vp, table[45:], lens[45:], vis[45:], got=first[45:])


@gpu
def test_as_many_sequences_and_nodes_as_are_served():
    lens = [(37 * i) % 49 - 1 for i in range(2048)]
    table, n = _table([m + 1 if m >= 0 else 0 for m in lens], 16, 24)
    kp, vp = (_cache(n, 1, 16, 64, torch.float16, s) for s in (26, 27))
    _check(_q(2048, 1, 4, 64, torch.float16), kp, vp, table, lens, _trees(2048, 1, 0))
    table, n = _table([1034], 16, 1)
    kp, vp = (_cache(n, 1, 16, 64, torch.float16, s) for s in (26, 27))
    _check(_q(1, 1024, 2, 64, torch.float16), kp, vp, table, [10], _trees(1, 1024, 0))


@gpu
def test_rope_append_slots():
    """Nodes are rotated by their depth and stored by their index."""
    from moeinfra_b200 import kernels

    H, KV, hd, page = 4, 2, 64, 16
    cos, sin = ref.rotary_table(64, hd)
    parents = [-1, 0, 0, 1, 1, -1]
    depth = [0, 1, 1, 2, 2, 0]
    lens = [20, 31]
    table, n = _table([m + 6 for m in lens], page, 2)
    qkv = torch.randn(12, (H + 2 * KV) * hd, generator=torch.Generator().manual_seed(1)).half().cuda()
    seq = torch.tensor([0] * 6 + [1] * 6, dtype=torch.int32, device="cuda")
    pos = torch.tensor([m + d for m in lens for d in depth], dtype=torch.int32, device="cuda")
    slot = torch.tensor([m + i for m in lens for i in range(6)], dtype=torch.int32, device="cuda")
    kp, vp = (torch.zeros(n, KV, page, hd, dtype=torch.float16, device="cuda") for _ in range(2))
    q = kernels.rope_append(qkv, cos.cuda(), sin.cuda(), pos, table.cuda(), kp, vp, H, seq_ids=seq,
                            slots=slot)
    kernels.check_device()
    wk, wv = torch.zeros_like(kp), torch.zeros_like(vp)
    for t in range(12):  # one token a call, at its slot through a table of its own
        where = torch.full((1, 64), -1, dtype=torch.int32, device="cuda")
        where[0, int(pos[t]) // page] = 0
        k1, v1 = (torch.zeros(1, KV, page, hd, dtype=torch.float16, device="cuda") for _ in range(2))
        want = kernels.rope_append(qkv[t:t + 1], cos.cuda(), sin.cuda(), pos[t:t + 1], where, k1, v1, H)
        assert torch.equal(q[t:t + 1], want)
        at, s = table[int(seq[t]), int(slot[t]) // page], int(slot[t]) % page
        wk[at, :, s], wv[at, :, s] = k1[0, :, int(pos[t]) % page], v1[0, :, int(pos[t]) % page]
    assert torch.equal(kp, wk) and torch.equal(vp, wv)
    assert len(parents) == 6
    for bad in (-1, 64):
        kernels.rope_append(qkv[:1], cos.cuda(), sin.cuda(), pos[:1], table.cuda(), kp, vp, H,
                            slots=torch.tensor([bad], dtype=torch.int32, device="cuda"))
        with pytest.raises(RuntimeError, match="out of range"):
            kernels.check_device()
    assert torch.equal(kp, wk) and torch.equal(vp, wv)


def test_tree_masks():
    from moeinfra_b200 import kernels

    assert kernels.tree_masks([]).shape == (0, 0)
    assert kernels.tree_masks([-1, 0, 0, 2]).tolist() == [[1], [3], [5], [13]]
    rng = random.Random(1)
    parents = _parents(rng, 200)
    bits = _bits(kernels.tree_masks(parents), 200)
    for i, p in enumerate(parents):
        want = bits[p].clone() if p >= 0 else torch.zeros(200, dtype=torch.bool)
        want[i] = True
        assert torch.equal(bits[i], want)
    for bad in ([0], [-1, 1], [-2]):
        with pytest.raises(ValueError, match="parent"):
            kernels.tree_masks(bad)


def test_refusals_on_the_host():
    from moeinfra_b200 import _native, kernels

    lib, fake = _native.lib(), 0x100000
    q, k = torch.zeros(2, 3, 4, 64, dtype=torch.float16), torch.zeros(3, 2, 16, 64, dtype=torch.float16)
    table, lens = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    vis = torch.zeros(2, 3, 1, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        kernels.tree_attention(q, k, k, table, lens, vis)

    def call(k=fake, ks=2048, n=3, kv=2, page=16, hd=64, dt=0, table=fake, ts=4, seqs=2, most=4, q=fake,
             qs=768, qn=256, nodes=3, heads=4, lengths=fake, visible=fake, vs=3, vn=1, scale=0.125, out=fake,
             ws=fake, nbytes=1 << 30):
        return lib.moe_tree_attention(_native.TREE_ATTENTION.pack(
            k, k, ks, ks, n, kv, page, hd, dt, table, ts, seqs, most, q, qs, qn, nodes, heads, lengths, 0,
            visible, vs, vn, scale, out, ws, nbytes, 0))

    assert lib.moe_tree_attention(None) == 1 and lib.moe_rope_append_slots(None, None) == 1
    assert call(heads=3) == 1 and call(heads=0) == 1 and call(nodes=-1) == 1 and call(scale=0.0) == 1
    assert call(scale=math.inf) == 1 and call(qn=255) == 1 and call(qs=0) == 1 and call(vs=-1) == 1
    assert call(q=0) == 1 and call(lengths=0) == 1 and call(visible=0) == 1 and call(out=0) == 1
    assert call(page=24, ks=4096) == 2 and call(seqs=2049) == 2 and call(nodes=1025) == 2
    assert call(hd=96, ks=4096) == 2 and call(most=(1 << 26) + 1, ts=1 << 27) == 2
    assert call(dt=2) == 2 and call(seqs=0) == 0 and call(nodes=0) == 0
    assert call(q=fake + 8) == 5 and call(qn=260) == 5 and call(visible=fake + 4) == 5
    assert call(ws=0) == 4 and call(nbytes=4096) == 4 and call(ws=fake + 8) == 5
    assert lib.moe_tree_attention_workspace_size(96) == 0


@gpu
def test_refusals_by_name():
    from moeinfra_b200 import kernels

    q = torch.zeros(2, 3, 4, 64, dtype=torch.float16, device="cuda")
    k = torch.zeros(3, 2, 16, 64, dtype=torch.float16, device="cuda")
    table = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    lens, vis = table[:, 0].contiguous(), torch.zeros(2, 3, 1, dtype=torch.int64, device="cuda")
    for args, name in (((q.float(), k, k, table, lens, vis), "q must be"),
                       ((q[:, :, :3].contiguous(), k, k, table, lens, vis), "do not divide"),
                       ((q, k, k[:2], table, lens, vis), "v_pages"),
                       ((q, k, k, table, lens.long(), vis), "lengths"),
                       ((q, k, k, table, lens, vis.int()), "visible"),
                       ((q, k, k, table, lens, vis[:, :2]), "visible"),
                       ((q, k, k, table, lens, vis, lens[:1]), "counts"),
                       ((q.cpu(), k, k, table, lens, vis), "q is on cpu"),
                       ((q, k[:, :, :15].contiguous(), k[:, :, :15].contiguous(), table, lens, vis),
                        "multiple of 16")):
        with pytest.raises((ValueError, RuntimeError), match=name):
            kernels.tree_attention(*args)
    with pytest.raises(ValueError, match="workspace"):
        kernels.tree_attention(q, k, k, table, lens, vis, workspace=torch.zeros(16, device="cuda"))
    with pytest.raises(ValueError, match="slots"):
        kernels.rope_append(torch.zeros(2, 8 * 64, device="cuda").half(), torch.zeros(8, 32, device="cuda"),
                            torch.zeros(8, 32, device="cuda"), lens, table, k, k.clone(), 4,
                            slots=lens.long())


@gpu
def test_rows_computed_again_outlast_no_wait():
    """Rows are computed again when no other warp waits for the one that does it: 32 rows of 8192 keys
    take longer than the 2 ms allowed here."""
    from moeinfra_b200 import _native, kernels

    # 300 units of 131 places over the SMs: every CTA has a whole one between two that are cut.
    seqs, nodes, H, hd, page, n = 300, 4, 16, 64, 64, 8188
    kp, vp = (_cache(128, 1, page, hd, torch.float16, s) for s in (1, 2))
    table = torch.arange(128, dtype=torch.int32).repeat(seqs, 1)
    q = _q(seqs, nodes, H, hd, torch.float16)
    visible = kernels.tree_masks([-1] * nodes)[None].expand(seqs, nodes, 1)
    at = torch.full((seqs,), n, dtype=torch.int32, device="cuda")
    args = (q.cuda(), kp, vp, table.cuda(), at, visible.cuda())
    clean = kernels.tree_attention(*args)
    _check(q[:2], kp, vp, table[:2], [n, n], visible[:2], got=clean[:2])
    vp[127, 0, page - 1, 7] = math.inf  # node 3's, which the other nodes do not see
    old = _native.wait_limit_ns()
    _native.set_wait_limit_ns(2_000_000)
    try:
        got = kernels.tree_attention(*args)
        kernels.check_device()
    finally:
        _native.set_wait_limit_ns(old)
    assert not got[:, 3, :, 7].isfinite().any()
    got[:, 3, :, 7] = clean[:, 3, :, 7]
    assert got.isfinite().all()
    # The same rows with probabilities rounded to 16 bits or not, and two results rounded: each by
    # 2^-11 of at most max |v| < 6.
    assert float((got.float() - clean.float()).abs().max()) <= 3 * 6 * 2.0 ** -11


@gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("seqs,lo", [(4, 100), (90, 100), (90, 700), (3, 5000)])
@pytest.mark.parametrize("nodes", [9, 40])
def test_rows_are_computed_again_in_every_form(seqs, lo, nodes, hd):
    """An infinity in a node that others do not see, in units of one tile and of two, that have a CTA each,
    lie whole between cuts, or are cut: the rows that do not see it are as without it."""
    from moeinfra_b200 import kernels

    H, KV, page = 8, 2, 16
    lens = [lo + 13 * i % 50 for i in range(seqs)]
    table, n = _table([m + nodes for m in lens], page, 8)
    kp, vp = (_cache(n, KV, page, hd, torch.float16, s) for s in (5, 6))
    q, visible = _q(seqs, nodes, H, hd, torch.float16), _trees(seqs, nodes, 2)
    at = torch.tensor(lens, dtype=torch.int32, device="cuda")
    args = (q.cuda(), kp, vp, table.cuda(), at, visible.cuda())
    clean = kernels.tree_attention(*args)
    _check(q[:2], kp, vp, table[:2], lens[:2], visible[:2], got=clean[:2])
    for b, m in enumerate(lens):
        vp[int(table[b, (m + 4) // page]), :, (m + 4) % page, hd - 1] = math.inf
    got = kernels.tree_attention(*args)
    kernels.check_device()
    sees = _bits(visible, nodes)[:, :, 4].cuda()
    assert not got[sees][..., hd - 1].isfinite().any()
    got[..., hd - 1] = torch.where(sees[..., None], clean[..., hd - 1], got[..., hd - 1])
    assert got.isfinite().all()
    # Probabilities rounded to 16 bits or not, and two results rounded: each by 2^-11 of at most
    # max |v| < 6.
    assert float((got.float() - clean.float()).abs().max()) <= 3 * 6 * 2.0 ** -11


@gpu
@pytest.mark.parametrize("H,KV,nodes", [(32, 8, 4), (32, 8, 1), (8, 2, 16), (8, 8, 9), (32, 8, 64)])
@pytest.mark.parametrize("seqs", [1, 5, 64])
def test_tables_wider_than_the_sequences(H, KV, nodes, seqs):
    """A table as wide as the longest sequence that may come, over short ones: the results are those of a
    table that ends with them, whichever kernel and cut its width picks."""
    from moeinfra_b200 import kernels

    lens, page, hd = [(29 * i) % 97 for i in range(seqs)], 16, 64
    narrow, n = _table([m + nodes for m in lens], page, 7)
    wide, _ = _table([m + nodes for m in lens], page, 7, width=2048 // page)
    kp, vp = (_cache(n, KV, page, hd, torch.bfloat16, s) for s in (1, 2))
    q, visible = _q(seqs, nodes, H, hd, torch.bfloat16), _trees(seqs, nodes, 5)
    for table in (narrow, wide):
        _check(q, kp, vp, table, lens, visible)


@gpu
@pytest.mark.parametrize("nodes,heads", [(3, 4), (9, 8)])
def test_a_result_over_the_queries_is_refused(nodes, heads):
    """A row may be computed again from its query after results were written.  A result between two
    sequences' queries is none over them."""
    from moeinfra_b200 import kernels

    k = _cache(4, 2, 16, 64, torch.float16, 1)
    table = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2)
    lens, vis = torch.full((2,), 5, dtype=torch.int32, device="cuda"), _trees(2, nodes, 1).cuda()
    buf = _q(8, nodes, heads, 64, torch.float16).cuda()
    want = kernels.tree_attention(buf[::7], k, k, table, lens, vis)
    for q, out in ((buf[:2], buf[:2]), (buf[:2], buf[1:3]), (buf[1:3], buf[:2]), (buf[::7], buf[6:8])):
        with pytest.raises(RuntimeError, match="status 1"):
            kernels.tree_attention(q, k, k, table, lens, vis, out=out)
    got = kernels.tree_attention(buf[::7], k, k, table, lens, vis, out=buf[3:5])
    assert got.data_ptr() == buf[3].data_ptr() and torch.equal(got, want)


@gpu
@pytest.mark.parametrize("nodes", [2, 20])
def test_a_table_of_two_to_the_30_positions(nodes):
    lens, page = [70000], 65536
    table, n = _table([lens[0] + nodes], page, 3, width=(1 << 30) // page)
    kp, vp = (_cache(n, 1, page, 64, torch.float16, s) for s in (1, 2))
    _check(_q(1, nodes, 4, 64, torch.float16), kp, vp, table, lens, _trees(1, nodes, 4))


def test_a_line_past_32_bits_is_refused():
    """Units times a table's steps; on the host, the pointers are never used."""
    from moeinfra_b200 import _native

    fake = 0x100000
    for seqs, kv, pages in ((128, 1, 1 << 14), (16, 8, 1 << 14), (2048, 8, 1 << 11)):  # of 65536
        assert _native.lib().moe_tree_attention(_native.TREE_ATTENTION.pack(
            fake, fake, kv << 22, kv << 22, 3, kv, 1 << 16, 64, 0, fake, pages, seqs, pages, fake,
            20 * 64 * 8, 64 * 8, 20, 8, fake, 0, fake, 20, 1, 0.125, 1 << 40, fake, 1 << 30, 0)) == 2
