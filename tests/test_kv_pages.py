"""fork_pages and keep_nodes: tables, lengths and counts equal the step-by-step oracle's, pages bit
for bit (nothing is computed, so no tolerance)."""
from __future__ import annotations

import random

import pytest
import torch

from oracle import branches

gpu = pytest.mark.gpu


def _state(rng, seqs, max_pages, page, kv=2, hd=64, layers=2, dtype=torch.float16, spare=0, most=None,
           extra_cols=0):
    """A consistent random state on the CPU: rows that share prefixes, counts, lengths."""
    rows, used = [], 0
    for i in range(seqs):
        n = rng.randint(0, most if most is not None else max_pages * page)
        need = -(-n // page)
        row = []
        if rows and rng.random() < 0.6:  # shares some pages of an earlier row
            src = rng.choice(rows)
            row = src[1][:rng.randint(0, min(need, -(-src[0] // page)))]
        while len(row) < need:
            row.append(used)
            used += 1
        rows.append((n, row))
    pool = used + spare
    order = list(range(pool))
    rng.shuffle(order)
    table = torch.full((seqs, max_pages + extra_cols), -1, dtype=torch.int32)
    refs = torch.zeros(pool, dtype=torch.int32)
    for i, (_, row) in enumerate(rows):
        for c, g in enumerate(row):
            table[i, c] = order[g]
            refs[order[g]] += 1
    g = torch.Generator().manual_seed(rng.randrange(1 << 30))
    shape = (layers, pool, kv, page, hd)
    k, v = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
    lengths = torch.tensor([n for n, _ in rows], dtype=torch.int32)
    return k, v, table, lengths, refs


def _parents(rng, seqs, end=0.2):
    return torch.tensor([-1 if rng.random() < end else rng.randrange(seqs) for _ in range(seqs)],
                        dtype=torch.int32)


def _equal(got, want):
    for name, x, y in zip(("k", "v", "table", "lengths", "refs"), got, want):
        assert torch.equal(x.cpu(), y), name


def _fork(state, parents, room):
    from moeinfra_b200 import kernels

    dev = [t.cuda() for t in state]
    kernels.fork_pages(*dev[:4], parents.cuda(), dev[4], room)
    kernels.check_device()
    return dev


@gpu
@pytest.mark.parametrize("seqs,max_pages,page,room", [
    (1, 1, 16, 1), (4, 5, 16, 1), (4, 5, 16, 0), (5, 3, 7, 9), (37, 9, 4, 6), (64, 40, 16, 1),
    (200, 33, 2, 70), (700, 3, 16, 1), (1500, 2, 1, 1)])
@pytest.mark.parametrize("seed", [0, 1])
def test_fork(seqs, max_pages, page, room, seed):
    rng = random.Random(1000 * seed + seqs)
    spare = seqs * (room // page + 2)
    state = _state(rng, seqs, max_pages, page, spare=spare)
    parents = _parents(rng, seqs)
    want = [t.clone() for t in state]
    assert branches.fork(*want[:4], parents, want[4], room)
    _equal(_fork(state, parents, room), want)


@gpu
@pytest.mark.parametrize("hd,dtype,kv,page", [(64, torch.bfloat16, 1, 48), (128, torch.float16, 3, 16),
                                               (128, torch.bfloat16, 8, 130)])
def test_fork_layouts(hd, dtype, kv, page):
    """Head sizes, odd pages, one layer as four dimensions, pages and rows further apart."""
    rng = random.Random(hd + kv)
    state = _state(rng, 6, 4, page, kv, hd, 1, dtype, spare=14, most=3 * page + 5)
    parents = torch.tensor([0, 0, 0, 5, 4, 5], dtype=torch.int32)
    want = [t.clone() for t in state]
    assert branches.fork(*want[:4], parents, want[4])
    from moeinfra_b200 import kernels

    k, v, table, lengths, refs = (t.cuda() for t in state)
    wide = torch.zeros(k.shape[1], 2, *k.shape[2:], dtype=dtype, device="cuda")
    wide[:, 0], wide[:, 1] = k[0], v[0]
    far = torch.full((6, 9), 77, dtype=torch.int32, device="cuda")
    far[:, 2:6] = table
    kernels.fork_pages(wide[:, 0], wide[:, 1], far[:, 2:6], lengths, parents.cuda(), refs)
    kernels.check_device()
    _equal((wide[None, :, 0], wide[None, :, 1], far[:, 2:6], lengths, refs), want)
    assert bool((far[:, :2] == 77).all()) and bool((far[:, 6:] == 77).all())


@gpu
def test_fork_of_a_held_prefix_leaves_it():
    """A page with a holder outside the table is copied by every row that writes there."""
    rng = random.Random(5)
    state = _state(rng, 4, 4, 16, spare=20, most=40)
    state[3][:] = 20
    state[2][:] = -1
    state[4].zero_()
    state[2][:, 0], state[2][:, 1] = 3, 7
    state[4][3] = state[4][7] = 4 + 1
    parents = torch.tensor([3, 2, 1, 0], dtype=torch.int32)
    want = [t.clone() for t in state]
    assert branches.fork(*want[:4], parents, want[4])
    assert int(want[4][7]) == 1 and int(want[4][3]) == 5
    _equal(_fork(state, parents, 1), want)


@gpu
def test_pages_freed_by_a_call_serve_it_and_none_left_is_reported():
    from moeinfra_b200 import _native, kernels

    k = torch.zeros(1, 3, 1, 16, 64, dtype=torch.float16)
    table = torch.tensor([[0, 1], [2, -1]], dtype=torch.int32)
    state = [k, k.clone(), table, torch.tensor([20, 4], dtype=torch.int32),
             torch.ones(3, dtype=torch.int32)]
    parents = torch.tensor([0, 0], dtype=torch.int32)  # row 1's page 2 is freed and taken again
    want = [t.clone() for t in state]
    assert branches.fork(*want[:4], parents, want[4])
    got = _fork(state, parents, 1)
    _equal(got, want)
    state[2] = torch.tensor([[0, 1], [0, 1]], dtype=torch.int32)
    state[4] = torch.tensor([2, 2, 1], dtype=torch.int32)  # page 2 is held elsewhere
    want = [t.clone() for t in state]
    assert not branches.fork(*want[:4], parents, want[4])
    dev = [t.cuda() for t in state]
    kernels.fork_pages(*dev[:4], parents.cuda(), dev[4])
    assert _native.stream_check(torch.cuda.current_stream().cuda_stream) == _native.MOE_ERR_PAGE
    _equal(dev, want)


@gpu
def test_bad_parents_lengths_and_pages_are_reported():
    from moeinfra_b200 import _native, kernels

    stream = torch.cuda.current_stream().cuda_stream
    for parents, length, entry in (([0, 2], 4, 0), ([0, 1], 33, 0), ([0, 1], 4, 3)):
        k = torch.zeros(1, 3, 1, 16, 64, dtype=torch.float16, device="cuda")
        table = torch.tensor([[entry, -1], [1, -1]], dtype=torch.int32, device="cuda")
        refs = torch.tensor([1, 1, 0], dtype=torch.int32, device="cuda")
        kernels.fork_pages(k, k.clone(), table,
                           torch.tensor([length, 4], dtype=torch.int32, device="cuda"),
                           torch.tensor(parents, dtype=torch.int32, device="cuda"), refs)
        assert _native.stream_check(stream) == _native.MOE_ERR_PAGE, (parents, length, entry)
    assert _native.stream_check(stream) == 0


@gpu
def test_fork_follows_its_inputs_in_a_graph_beside_another():
    """Two captured calls on one stream, replayed on two at once: each has its own scratch."""
    from moeinfra_b200 import kernels

    rng = random.Random(11)
    states = [_state(rng, 24, 6, 16, spare=60) for _ in range(2)]
    dev = [[t.cuda() for t in s] for s in states]
    par = [torch.zeros(24, dtype=torch.int32, device="cuda") for _ in range(2)]
    kernels.fork_pages(*[t.clone() for t in dev[0][:4]], par[0], dev[0][4].clone())
    graphs = []
    for d, p in zip(dev, par):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kernels.fork_pages(*d[:4], p, d[4])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(3):
        picks = [_parents(rng, 24) for _ in range(2)]
        for p, pick in zip(par, picks):
            p.copy_(pick)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for s, d, pick in zip(states, dev, picks):
            assert branches.fork(*s[:4], pick, s[4])
            _equal(d, s)
    kernels.check_device()


def _keep_state(rng, seqs, nodes, page, kv, hd, layers, dtype, hi=50):
    lens = [rng.randint(0, hi) for _ in range(seqs)]
    need = [-(-(n + nodes) // page) for n in lens]
    order = list(range(sum(need) + 2))
    rng.shuffle(order)
    table = torch.full((seqs, max(need) + 1), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    g = torch.Generator().manual_seed(rng.randrange(1 << 30))
    shape = (layers, sum(need) + 2, kv, page, hd)
    k, v = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
    keep = torch.full((seqs, nodes), -1, dtype=torch.int32)
    for b in range(seqs):
        path = sorted(rng.sample(range(nodes), rng.randint(0, nodes)))
        keep[b, :len(path)] = torch.tensor(path, dtype=torch.int32)
    return k, v, table, torch.tensor(lens, dtype=torch.int32), keep


@gpu
@pytest.mark.parametrize("seqs,nodes,page,kv,hd,layers,dtype", [
    (1, 1, 16, 1, 64, 1, torch.float16), (3, 16, 16, 8, 128, 3, torch.float16),
    (7, 33, 5, 3, 64, 2, torch.bfloat16), (2, 300, 64, 2, 128, 2, torch.bfloat16),
    (65, 4, 1, 1, 128, 1, torch.float16)])
def test_keep_nodes(seqs, nodes, page, kv, hd, layers, dtype):
    from moeinfra_b200 import kernels

    k, v, table, lengths, keep = _keep_state(random.Random(nodes), seqs, nodes, page, kv, hd, layers,
                                             dtype)
    lengths[-1] = -1 if seqs > 1 else lengths[-1]
    dk, dv = k.cuda(), v.cuda()
    wide = torch.full((seqs, nodes + 3), 10 ** 6, dtype=torch.int32, device="cuda")
    wide[:, :nodes] = keep.cuda()
    got = kernels.keep_nodes(dk, dv, table.cuda(), lengths.cuda(), wide[:, :nodes])
    kernels.check_device()
    assert got.tolist() == branches.keep_nodes(k, v, table, lengths, keep)
    assert torch.equal(dk.cpu(), k) and torch.equal(dv.cpu(), v)


@gpu
def test_keep_nodes_ends_a_list_at_its_first_bad_entry():
    from moeinfra_b200 import _native, kernels

    k, v, table, lengths, _ = _keep_state(random.Random(3), 3, 8, 16, 2, 64, 2, torch.float16)
    stream = torch.cuda.current_stream().cuda_stream
    for entry, cut in (([0, 3, 2, 5], 2), ([1, 1, 4, -1], 1), ([2, 4, 900, -1], 2)):
        keep = torch.tensor([entry] * 3, dtype=torch.int32)
        dk, dv = k.cuda(), v.cuda()
        got = kernels.keep_nodes(dk, dv, table.cuda(), lengths.cuda(), keep.cuda())
        assert _native.stream_check(stream) == _native.MOE_ERR_PAGE, entry
        wk, wv = k.clone(), v.clone()
        want = branches.keep_nodes(wk, wv, table, lengths, keep[:, :cut])
        assert got.tolist() == want and torch.equal(dk.cpu(), wk) and torch.equal(dv.cpu(), wv)
    after = torch.tensor([[0, -1, 10 ** 9]] * 3, dtype=torch.int32, device="cuda")
    kernels.keep_nodes(k.cuda(), v.cuda(), table.cuda(), lengths.cuda(), after)
    assert _native.stream_check(stream) == 0  # what follows the end is not looked at


@gpu
def test_nothing_to_do():
    from moeinfra_b200 import kernels

    k = torch.zeros(2, 3, 1, 16, 64, dtype=torch.float16, device="cuda")

    def i32(*shape):
        return torch.zeros(shape, dtype=torch.int32, device="cuda")

    kernels.fork_pages(k, k, i32(0, 4), i32(0), i32(0), i32(3))
    kernels.fork_pages(k, k, i32(4, 0), i32(4), i32(4), i32(3))
    assert kernels.keep_nodes(k, k, i32(0, 4), i32(0), i32(0, 5)).numel() == 0
    assert kernels.keep_nodes(k, k, i32(2, 4), i32(2) + 9, i32(2, 0)).tolist() == [9, 9]
    kernels.check_device()


def test_wrappers_refuse_what_the_kernels_cannot_take():
    """On the host, before any launch."""
    from moeinfra_b200 import kernels

    k = torch.zeros(2, 3, 1, 16, 64, dtype=torch.float16)
    i32 = torch.zeros(2, dtype=torch.int32)
    table = torch.zeros(2, 4, dtype=torch.int32)
    refs = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        kernels.fork_pages(k, k, table, i32, i32, refs)
    with pytest.raises(RuntimeError, match="no CPU path"):
        kernels.keep_nodes(k, k, table, i32, table)
    with pytest.raises(ValueError, match="k_pages must be"):
        kernels.fork_pages(k[0, 0], k, table, i32, i32, refs)
    with pytest.raises(ValueError, match="v_pages must have"):
        kernels.keep_nodes(k, k[:1], table, i32, table)
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        kernels.keep_nodes(k.float(), k.float(), table, i32, table)


@gpu
def test_wrappers_refuse_by_name():
    from moeinfra_b200 import kernels

    k = torch.zeros(2, 3, 1, 16, 64, dtype=torch.float16, device="cuda")
    i32 = torch.zeros(2, dtype=torch.int32, device="cuda")
    table = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    refs = torch.zeros(3, dtype=torch.int32, device="cuda")
    for name, args in (("lengths", (k, k, table, i32.long(), i32, refs)),
                       ("parents", (k, k, table, i32, i32[:1], refs)),
                       ("refs", (k, k, table, i32, i32, refs[:2])),
                       ("refs", (k, k, table, i32, i32, refs.cpu())),
                       ("block_table", (k, k, table.long(), i32, i32, refs)),
                       ("rows overlap", (k, k, table[:1].expand(2, 4), i32, i32, refs)),
                       ("layers overlap", (k[:1].expand(2, *k.shape[1:]), k, table, i32, i32, refs)),
                       ("head_dim", (k[..., :32].contiguous(),) * 2 + (table, i32, i32, refs))):
        with pytest.raises((ValueError, RuntimeError), match=name):
            kernels.fork_pages(*args)
    with pytest.raises(RuntimeError, match="status 1"):
        kernels.fork_pages(k, k, table, i32, i32, refs, room=-1)
    with pytest.raises(ValueError, match="workspace"):
        kernels.fork_pages(k, k, table, i32, i32, refs, workspace=refs)
    with pytest.raises(ValueError, match="keep"):
        kernels.keep_nodes(k, k, table, i32, i32)


def test_library_refuses_before_any_launch():
    """Pointers below are never used: the checks come first."""
    from moeinfra_b200 import _native

    lib = _native.lib()
    fake = 0x100000

    def kv(**over):
        f = dict(k=fake, v=fake, ks=2048, vs=2048, n=3, kv=2, page=16, hd=64, dt=0, table=fake, ts=4,
                 seqs=2, most=4) | over
        return list(f.values())

    def fork(layers=2, kl=6144, vl=6144, room=1, ws=fake, nbytes=1 << 20, lengths=fake, **over):
        return lib.moe_fork_pages(_native.FORK_PAGES.pack(
            *kv(**over), layers, kl, vl, lengths, fake, fake, room, ws, nbytes, 0))

    def keep(layers=2, kl=6144, vl=6144, stride=5, most=5, lengths=fake, **over):
        return lib.moe_keep_nodes(_native.KEEP_NODES.pack(
            *kv(**over), layers, kl, vl, lengths, fake, stride, most, fake, 0))

    for call in (fork, keep):
        assert call(layers=0) == 1 and call(kl=-8) == 1 and call(kl=4) == 5
        assert call(dt=2) == 2 and call(hd=96) == 2 and call(ks=8) == 1 and call(k=fake + 2) == 5
        assert call(lengths=0) == 1 and call(seqs=-1) == 1 and call(ts=3) == 1
        assert call(seqs=0) == 0
        assert call(n=1 << 40) == 2
    assert fork(room=-1) == 1 and fork(seqs=8193) == 2 and fork(most=0) == 0
    assert fork(nbytes=4096) == 4 and fork(ws=fake + 8) == 5 and fork(ws=0) == 4
    assert keep(most=6) == 1 and keep(most=-1) == 1
    assert lib.moe_fork_pages(None) == 1 and lib.moe_keep_nodes(None) == 1
    assert lib.moe_fork_pages_workspace_size(-1) == 0 and lib.moe_fork_pages_workspace_size(9000) == 0


def test_the_oracle_keeps_its_counts():
    """Counts equal the table's entries after any sequence of forks, and no two rows write one page."""
    rng = random.Random(2)
    state = _state(rng, 12, 6, 4, kv=1, layers=1, spare=60)
    for _ in range(20):
        parents = _parents(rng, 12)
        assert branches.fork(*state[:4], parents, state[4], 3)
        table, lengths, refs = state[2:]
        held = torch.zeros_like(refs)
        for g in table.flatten().tolist():
            if g >= 0:
                held[g] += 1
        assert torch.equal(held, refs)
        for i, n in enumerate(lengths.tolist()):
            if parents[i] >= 0 and n // 4 < 6:
                assert int(refs[table[i, n // 4]]) == 1


@gpu
@pytest.mark.parametrize("seqs,max_pages,page,room", [(6, 5, 16, 1), (5, 3, 7, 0), (40, 40, 16, 20),
                                                       (300, 3, 4, 9), (1500, 2, 1, 1)])
def test_fork_passes_over_rows_without_a_sequence(seqs, max_pages, page, room):
    """Rows of a negative length stay so, as do their copies; neither is given a page."""
    rng = random.Random(seqs)
    state = _state(rng, seqs, max_pages, page, spare=seqs * (room // page + 2))
    idle = torch.tensor([rng.random() < 0.4 for _ in range(seqs)])
    idle[0], idle[1] = True, False
    state[3][idle] = torch.tensor([rng.choice([-1, -1, -7, -2 ** 31]) for _ in range(seqs)],
                                  dtype=torch.int32)[idle]
    for b in range(0, seqs, 2):  # half of them hold no pages
        if idle[b]:
            for g in state[2][b].tolist():
                if g >= 0:
                    state[4][g] -= 1
            state[2][b] = -1
    for parents in (torch.arange(seqs, dtype=torch.int32), torch.zeros(seqs, dtype=torch.int32),
                    _parents(rng, seqs)):
        want = [t.clone() for t in state]
        assert branches.fork(*want[:4], parents, want[4], room)
        assert torch.equal(want[3], torch.where(parents >= 0, state[3][parents.clamp(min=0).long()], 0))
        got = _fork(state, parents, room)
        _equal(got, want)
        none = want[3] < 0
        assert torch.equal(want[2][none], state[2][parents[none].long()])


def test_new_lengths_over_the_old_ones_are_refused():
    """The CTAs of a sequence read its length while one writes the new one.  On the host; the pointers are
    never used."""
    from moeinfra_b200 import _native

    fake = 0x100000

    def keep(lengths, new, seqs=3):
        return _native.lib().moe_keep_nodes(_native.KEEP_NODES.pack(
            fake, fake, 2048, 2048, 3, 2, 16, 64, 0, fake, 4, seqs, 4, 1, 0, 0, lengths, fake, 5, 5, new, 0))

    for new in (fake, fake + 8, fake - 8):
        assert keep(fake, new) == 1, new


@gpu
@pytest.mark.parametrize("max_pages", [2, 3])
def test_as_many_rows_as_fork(max_pages):
    """8192 rows, their table in one CTA's shared memory and in two CTAs'."""
    rng = random.Random(max_pages)
    state = _state(rng, 8192, max_pages, 2, kv=1, layers=1, spare=8192)
    parents = _parents(rng, 8192)
    want = [t.clone() for t in state]
    assert branches.fork(*want[:4], parents, want[4])
    _equal(_fork(state, parents, 1), want)
