"""Beams and drafted trees through the engine: the operators run together, as a generation uses them.

Numbers are compared where the model is continuous (a stand-in MoE), with the tolerance of
``test_paged_engine``: two arithmetics of one stack differ by up to 5e-3 of the logits' norm, derived
there.  A log-probability then differs by at most twice that.
"""
from __future__ import annotations

import random
from types import SimpleNamespace

import pytest
import torch

from tests.test_engine_gpu import V, _config, ckpt  # noqa: F401 (fixture)
from tests.test_paged_engine import PAGED, LinearMoE, _ragged

gpu = pytest.mark.gpu
CLOSE = 5e-3


def _stack(heads=4, kv=2, hd=64, seed=5, max_batch=8, max_len=160, page=16, pages=None):
    from moeinfra_b200.engine.dense import DenseConfig
    from moeinfra_b200.engine.paged import PagedDenseStack
    from moeinfra_b200.model.types import LayerWeights

    hidden, layers, vocab, g = 256, 2, 512, torch.Generator().manual_seed(seed)

    def r(*shape):
        return torch.randn(*shape, generator=g) * 0.05

    weights = [LayerWeights(1 + r(hidden), r(heads * hd, hidden), r(kv * hd, hidden),
                            r(kv * hd, hidden), r(hidden, heads * hd), 1 + r(hidden),
                            torch.zeros(8, hidden)) for _ in range(layers)]
    moes = [LinearMoE(r(hidden, hidden).half().cuda()) for _ in range(layers)]
    return PagedDenseStack(DenseConfig(hidden, heads, kv, hd, vocab, 1e6, 1e-5), weights,
                           4 * r(vocab, hidden), 1 + r(hidden), 3 * r(vocab, hidden), moes, "cuda",
                           max_batch=max_batch, max_len=max_len, page_size=page, num_pages=pages)


def _logits_after(stack, seqs):
    """fp32 logits after whole sequences, by prefill alone."""
    out = []
    for i in range(0, len(seqs), stack.max_batch):
        part = [torch.tensor(s) for s in seqs[i:i + stack.max_batch]]
        stack.cache.reserve([len(s) for s in part])
        out.append(stack.prefill(part).float())
    return torch.cat(out)


@gpu
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("heads,kv,hd", [(4, 2, 64), (4, 1, 128)])
@torch.no_grad()
def test_beam_steps_find_what_recomputed_sequences_score(heads, kv, hd, captured):
    """The forked cache's scores are those of the sequences computed from scratch, at every step, and
    no continuation of a kept beam scores above the kept ones."""
    from moeinfra_b200 import kernels
    from moeinfra_b200.engine.engine import _BeamStep

    B, K, steps = 2, 3, 20  # 20 steps cross a page of 16 twice
    stack, plain = _stack(heads, kv, hd), _stack(heads, kv, hd)
    rows = [r.tolist() for r in _ragged([14, 33])[0]]
    step = _BeamStep(SimpleNamespace(_device=stack.device, _stack=stack), B, K)
    stack.cache.clear()
    if captured:
        step.capture()
        stack.cache.clear()
    stack.cache.reserve([len(rows[0]), 0, 0, len(rows[1]), 0, 0])
    logits = stack.prefill([torch.tensor(r) for r in rows], stride=K)
    first = step.begin(logits, stack.prompt_lengths)
    paths = [[rows[b] + [t] for t in first[b].tolist()] for b in range(B)]
    exact = torch.log_softmax(_logits_after(plain, rows), -1)
    score = torch.stack([exact[b][first[b]] for b in range(B)]).cpu()
    off = 2 * CLOSE * float(logits.float().norm(dim=-1).max())
    best = exact.topk(K).values.cpu()
    assert float((score - best).abs().max()) <= off
    for i in range(1, steps):
        step.run()
        tokens, parents = step.ids.view(B, K).tolist(), step.parents.tolist()
        full = _logits_after(plain, [p for b in range(B) for p in paths[b]])
        off += 2 * CLOSE * float(full.norm(dim=-1).max())
        every = score[:, :, None] + torch.log_softmax(full, -1).view(B, K, -1).cpu()
        for b in range(B):
            picks = [float(every[b, p, t]) for p, t in zip(parents[b], tokens[b])]
            best = every[b].flatten().topk(K).values
            for j in range(K):  # as good as the best ones, within what both may be off
                assert picks[j] >= float(best[j]) - 2 * off
                assert abs(float(step.scores[b, j]) - picks[j]) <= off
            score[b] = torch.tensor(picks)
            paths[b] = [paths[b][p] + [t] for p, t in zip(parents[b], tokens[b])]
            assert len({tuple(p) for p in paths[b]}) == K
        assert step.lengths.tolist() == [len(rows[b]) + i for b in range(B) for _ in range(K)]
    kernels.check_device()
    table, refs = stack.cache.block_table, stack.cache.refs
    held = torch.bincount(table[table >= 0].long(), minlength=len(refs))
    assert torch.equal(held.int(), refs)
    # The prompts' full pages are still shared by their beams.
    assert int(refs[table[0, 0]]) >= (K if len(rows[0]) >= 16 else 1) and int(refs[table[3, 0]]) == K


@gpu
@pytest.mark.parametrize("heads,kv,hd,page", [(4, 2, 64, 16), (4, 4, 128, 32), (7, 1, 64, 48)])
@torch.no_grad()
def test_verified_trees_continue_as_decoding_does(heads, kv, hd, page):
    """Trees around a given continuation: verify, accept the nodes on it, go on behind them.  The
    logits after each accepted node are those of decoding the same tokens one by one."""
    from moeinfra_b200 import kernels

    rng = random.Random(hd + page)
    stack, plain = _stack(heads, kv, hd, page=page), _stack(heads, kv, hd, page=page)
    rows = [r.tolist() for r in _ragged([12, 1, 40])[0]]
    B, total, T = len(rows), 30, 11
    tail = [[rng.randrange(512) for _ in range(total + T)] for _ in range(B)]
    stack.cache.reserve([len(r) + total + 2 * T for r in rows])
    stack.prefill([torch.tensor(r) for r in rows])
    plain.cache.reserve([len(r) + total + T for r in rows])
    plain.prefill([torch.tensor(r) for r in rows])
    pos = torch.tensor([len(r) for r in rows], dtype=torch.int32, device="cuda")
    want = []
    for i in range(total + T):
        ids = torch.tensor([t[i] for t in tail], device="cuda")[:, None]
        want.append(plain.decode(ids, pos).float())
        pos += 1
    lengths = torch.tensor([len(r) for r in rows], dtype=torch.int32, device="cuda")
    done, steps = [0] * B, 0
    while min(done) < total:
        ids, masks, depths, keep = [], [], [], []
        for b in range(B):
            parents = [-1] + [rng.randint(max(0, j - 4), j - 1) for j in range(1, T)]
            depth = [0]
            for p in parents[1:]:
                depth.append(depth[p] + 1)
            on, token = [0], [tail[b][done[b]]]
            for j in range(1, T):  # a node on the path so far may carry the next token
                real = parents[j] == on[-1] and rng.random() < 0.7
                token.append(tail[b][done[b] + depth[j]] if real else rng.randrange(512))
                if real:
                    on.append(j)
            ids.append(token)
            masks.append(kernels.tree_masks(parents))
            depths.append(depth)
            keep.append(on + [-1] * (T - len(on)))
        logits = stack.verify(torch.tensor(ids, device="cuda"), lengths,
                              torch.tensor(depths, dtype=torch.int32, device="cuda"),
                              torch.stack(masks).cuda()).float()
        for b in range(B):
            for d, node in enumerate(x for x in keep[b] if x >= 0):
                y = want[done[b] + d][b]
                assert float((logits[b, node] - y).norm() / y.norm()) < CLOSE, (b, steps, d)
        lengths = stack.accept(lengths, torch.tensor(keep, dtype=torch.int32, device="cuda"))
        for b in range(B):
            done[b] = min(done[b] + sum(x >= 0 for x in keep[b]), total)
            if done[b] == total:  # this sequence stays where it is
                lengths[b] = len(rows[b]) + total
        steps += 1
    kernels.check_device()
    assert steps < total
    # Behind the trees plain decoding goes on over the compacted cache.
    ids = torch.tensor([t[total] for t in tail], device="cuda")[:, None]
    got = stack.decode(ids, lengths).float()
    for b in range(B):
        y = want[total][b]
        assert float((got[b] - y).norm() / y.norm()) < CLOSE


@gpu
@torch.no_grad()
def test_verify_passes_over_rows_without_a_sequence():
    from moeinfra_b200 import kernels

    stack = _stack()
    rows = _ragged([12, 20])[0]
    stack.cache.reserve([40, 40])
    stack.prefill([r.clone() for r in rows])
    lengths = torch.tensor([12, -1], dtype=torch.int32, device="cuda")
    ids = torch.tensor([[5, 6, 7, 8]] * 2, device="cuda")
    depths = torch.tensor([0, 1, 1, 2], dtype=torch.int32, device="cuda")
    visible = kernels.tree_masks([-1, 0, 0, 2]).cuda()
    own = stack.cache.block_table[1][stack.cache.block_table[1] >= 0].long()
    before = [p[:, own].clone() for p in (stack.cache.k_pages, stack.cache.v_pages)]
    logits = stack.verify(ids, lengths, depths, visible)
    kernels.check_device()
    for pages, was in zip((stack.cache.k_pages, stack.cache.v_pages), before):
        assert torch.equal(pages[:, own], was)
    alone = stack.verify(ids[:1], lengths[:1], depths, visible)
    assert float((logits[0] - alone[0]).float().norm() / alone.float().norm()) < CLOSE
    keep = torch.tensor([[0, 2], [0, 2]], dtype=torch.int32, device="cuda")
    assert stack.accept(lengths, keep).tolist() == [14, -1]
    for pages, was in zip((stack.cache.k_pages, stack.cache.v_pages), before):
        assert torch.equal(pages[:, own], was)
    kernels.check_device()


def _beams(cfg, ids, mask, n, beams):
    from moeinfra_b200.engine.engine import InferenceEngine
    from moeinfra_b200.engine.types import ForwardRequest

    with InferenceEngine(cfg) as eng:
        return eng.generate(ForwardRequest(ids, mask, n, num_beams=beams))


@gpu
def test_engine_searches_with_beams(ckpt):  # noqa: F811
    """Graph and eager steps, one request after another, other requests between."""
    from moeinfra_b200.engine.engine import InferenceEngine
    from moeinfra_b200.engine.types import ForwardRequest

    over = PAGED | {"max_batch": 8}
    _, ids, mask = _ragged([12, 33])
    a = _beams(_config(ckpt, engine=over), ids, mask, 20, 4)
    b = _beams(_config(ckpt, engine=over | {"cuda_graphs": False}), ids, mask, 20, 4)
    assert a.token_ids == b.token_ids and a.scores == b.scores
    assert a.stage_timings["cuda_graph_decode"] and not b.stage_timings["cuda_graph_decode"]
    assert [len(t) for t in a.token_ids] == [20, 20] and all(s < 0 for s in a.scores)
    with InferenceEngine(_config(ckpt, engine=over)) as eng:
        greedy = eng.generate(ForwardRequest(ids, mask, 20)).token_ids
        c = eng.generate(ForwardRequest(ids, mask, 20, num_beams=4))
        d = eng.generate(ForwardRequest(ids, mask, 20, num_beams=3))
        assert eng.generate(ForwardRequest(ids, mask, 20)).token_ids == greedy
        e = eng.generate(ForwardRequest(ids, mask, 20, num_beams=4))
        one = eng.generate(ForwardRequest(ids, mask, 1, num_beams=4))
    assert c.token_ids == e.token_ids == a.token_ids and c.scores == e.scores
    assert len(d.token_ids) == 2 and [len(t) for t in one.token_ids] == [1, 1]
    assert [t[0] for t in greedy] == [t[0] for t in one.token_ids]


@gpu
def test_beams_fit_the_pool_they_need(ckpt):  # noqa: F811
    """Two prompts of 33 tokens and 4 beams of 15 more: 2 shared pages and one or two a beam, not the
    24 pages that 8 sequences of 48 hold."""
    _, ids, mask = _ragged([33, 33])
    need = 2 * (2 + 4 * (47 // 16 + 1 - 2))
    full = _beams(_config(ckpt, engine=PAGED | {"max_batch": 8}), ids, mask, 15, 4)
    tight = _beams(_config(ckpt, engine=PAGED | {"max_batch": 8, "kv_pages": need}), ids, mask, 15, 4)
    assert tight.token_ids == full.token_ids and need < 24
    with pytest.raises(RuntimeError, match="may be needed"):
        _beams(_config(ckpt, engine=PAGED | {"max_batch": 8, "kv_pages": need - 1}), ids, mask, 15, 4)


@gpu
def test_beam_request_checks(ckpt):  # noqa: F811
    from moeinfra_b200.engine.types import SamplingParams
    from moeinfra_b200.engine.engine import InferenceEngine
    from moeinfra_b200.engine.types import ForwardRequest

    ids = torch.zeros(2, 4, dtype=torch.long)
    with InferenceEngine(_config(ckpt, engine=PAGED | {"max_batch": 4})) as eng:
        for bad in (dict(num_beams=0), dict(num_beams=65), dict(num_beams=3), dict(num_beams=-2),
                    dict(num_beams=2, max_new_tokens=0), dict(num_beams=2, max_new_tokens=70),
                    dict(num_beams=2, sampling=SamplingParams())):
            with pytest.raises(ValueError):
                eng.generate(ForwardRequest(ids, **({"max_new_tokens": 2} | bad)))
        assert len(eng.generate(ForwardRequest(ids[:1], None, 2, num_beams=4)).token_ids) == 2
    with pytest.raises(ValueError, match="paged_kv"):
        _beams(_config(ckpt), ids, None, 2, 2)


def test_cache_counts_its_pages():
    """Host side of the counts (CPU)."""
    from moeinfra_b200.engine.paged import PagedKVCache

    c = PagedKVCache(1, 5, 1, 16, 64, max_batch=3, max_len=64, device="cpu")
    c.reserve([17, 0, 33])
    assert c.refs.tolist() == [1] * 5
    c.reserve([16])
    assert sorted(c.refs.tolist()) == [0, 0, 0, 0, 1] and int(c.refs[c.block_table[0, 0]]) == 1
    c.clear()
    assert c.free_pages == 5 and not c.refs.any() and bool((c.block_table == -1).all())


@gpu
@pytest.mark.parametrize("K,max_batch", [(2, 2), (4, 4), (2, 4)])
def test_beams_reach_the_cache_s_last_position(ckpt, K, max_batch):  # noqa: F811
    """The default pool holds max_batch sequences of max_seq_len, so it does for their beams: the
    position behind the last one has no page and needs none."""
    prompts = max_batch // K
    _, ids, mask = _ragged([5] * prompts)
    over = PAGED | {"max_batch": max_batch}          # 64 positions in pages of 16
    a = _beams(_config(ckpt, engine=over), ids, mask, 60, K)
    b = _beams(_config(ckpt, engine=over | {"kv_pages": 40}), ids, mask, 60, K)
    assert a.token_ids == b.token_ids and a.scores == b.scores
    rows = a.token_ids if prompts > 1 else [a.token_ids]
    assert [len(t) for t in rows] == [60] * prompts
    _, ids, mask = _ragged([64] * prompts)           # a prompt that fills its table
    one = _beams(_config(ckpt, engine=over), ids, mask, 1, K)
    assert len(one.scores) == prompts


@gpu
@pytest.mark.parametrize("over", [{}, {"num_beams": 2}, {"seed": 1}])
@pytest.mark.parametrize("paged", [True, False])
def test_a_result_s_logits_stay(ckpt, paged, over):  # noqa: F811
    """The next request of the same kind does not write into a result that the caller still holds."""
    from moeinfra_b200.engine.engine import InferenceEngine
    from moeinfra_b200.engine.types import ForwardRequest, SamplingParams

    if over.get("num_beams") and not paged:
        pytest.skip("beams need pages")
    kind = {"sampling": SamplingParams(**over)} if "seed" in over else over
    first, second = (torch.randint(0, V, (2, 9), generator=torch.Generator().manual_seed(s)) for s in (1, 2))
    with InferenceEngine(_config(ckpt, engine=(PAGED if paged else {}) | {"max_batch": 4})) as eng:
        a = eng.generate(ForwardRequest(first, None, 5, **kind))
        held = a.logits.clone()
        b = eng.generate(ForwardRequest(second, None, 5, **kind))
        assert a.stage_timings["cuda_graph_decode"]
        assert torch.equal(a.logits, held) and not torch.equal(a.logits, b.logits)


@gpu
def test_beam_logits_are_the_returned_sequences_(ckpt):  # noqa: F811
    """[prompts, 1, vocab] for any number of tokens: what each sequence's last token was chosen from."""
    from moeinfra_b200.engine.engine import InferenceEngine
    from moeinfra_b200.engine.types import ForwardRequest

    _, ids, mask = _ragged([12, 33])
    with InferenceEngine(_config(ckpt, engine=PAGED | {"max_batch": 8})) as eng:
        one = eng.generate(ForwardRequest(ids, mask, 1, num_beams=4))
        greedy = eng.generate(ForwardRequest(ids, mask, 1))
        assert one.logits.shape == (2, 1, V) and torch.equal(one.logits, greedy.logits)
        for n in (2, 9):
            many = eng.generate(ForwardRequest(ids, mask, n, num_beams=4))
            assert many.logits.shape == (2, 1, V)
            step = eng._graphs[2, 4, "beams"][1]
            rows = step.logits.view(2, 4, V)
            for b in range(2):
                assert torch.equal(many.logits[b, 0], rows[b, int(step.parents[b, 0])])


@gpu
@pytest.mark.parametrize("heads,kv,hd", [(4, 2, 64), (4, 1, 128)])
@torch.no_grad()
def test_forked_beams_are_what_recomputed_sequences_are(heads, kv, hd):
    """At every step the logits over the forked cache are those of each beam's own sequence computed from
    scratch, row by row and without what earlier steps were off, and the step's choice is the
    definition's for its own logits and scores."""
    from moeinfra_b200 import kernels
    from moeinfra_b200.engine.engine import _BeamStep
    from oracle import branches
    from tests.test_beam_select import _off

    B, K, steps = 2, 3, 36  # three page crossings of 16
    stack, plain = _stack(heads, kv, hd), _stack(heads, kv, hd)
    rows = [r.tolist() for r in _ragged([14, 33])[0]]
    step = _BeamStep(SimpleNamespace(_device=stack.device, _stack=stack), B, K)
    stack.cache.clear()
    stack.cache.reserve([len(rows[0]), 0, 0, len(rows[1]), 0, 0])
    first = step.begin(stack.prefill([torch.tensor(r) for r in rows], stride=K), stack.prompt_lengths)
    paths = [[rows[b] + [t] for t in first[b].tolist()] for b in range(B)]
    forks = 0
    for i in range(1, steps):
        before = step.scores.clone().cpu()
        logits = step.run()
        full = _logits_after(plain, [p for b in range(B) for p in paths[b]])
        err = (logits.float() - full).norm(dim=-1) / full.norm(dim=-1)
        assert float(err.max()) < CLOSE, (i, err.tolist())
        tokens, parents = step.ids.view(B, K).tolist(), step.parents.tolist()
        x = logits.double().cpu().view(B, K, -1)
        for b in range(B):
            want = branches.beam_select(logits.view(B, K, -1)[b].cpu(), before[b], K)[0]
            every = before[b].double()[:, None] + torch.log_softmax(x[b], -1)
            for j, (p, t) in enumerate(zip(parents[b], tokens[b])):
                v = float(every[p, t])
                off = _off(v, float(before[b, p]))
                assert abs(v - float(want[j])) <= 2 * off and abs(v - float(step.scores[b, j])) <= off
            forks += len(set(parents[b])) < K
            paths[b] = [paths[b][p] + [t] for p, t in zip(parents[b], tokens[b])]
            assert len({tuple(p) for p in paths[b]}) == K
    assert forks > 0  # rows were shared and copied, not only carried on
    kernels.check_device()


@gpu
@pytest.mark.parametrize("captured", [False, True])
@torch.no_grad()
def test_trees_grow_their_pages_beside_an_idle_row(captured):
    """A step is fork (each row its own parent, room for a tree), verify, accept, captured or not: pages come
    as they are needed, the row without a sequence gets none, and the logits are those of decoding."""
    from moeinfra_b200 import kernels

    rng = random.Random(17)
    stack, plain = _stack(), _stack()
    rows = [r.tolist() for r in _ragged([12, 1, 40])[0]]
    lens, T, steps = [12, -1, 1, 40], 6, 9  # row 1 is idle
    live = [b for b, n in enumerate(lens) if n >= 0]
    tail = {b: [rng.randrange(512) for _ in range(steps * T + 1)] for b in live}
    plain.cache.reserve([len(r) + steps * T + 1 for r in rows])
    plain.prefill([torch.tensor(r) for r in rows])
    pos = torch.tensor([len(r) for r in rows], dtype=torch.int32, device="cuda")
    want = []
    for i in range(steps * T):
        ids = torch.tensor([tail[b][i] for b in live], device="cuda")[:, None]
        want.append(dict(zip(live, plain.decode(ids, pos).float())))
        pos += 1
    cache = stack.cache
    cache.clear()

    def prompts():
        cache.reserve([max(n, 0) for n in lens])
        for b, r in zip(live, rows):  # one after the other, each in its own row of the table
            alone = stack.cache.block_table
            stack.cache.block_table = alone[b:b + 1]
            stack.prefill([torch.tensor(r)])
            stack.cache.block_table = alone

    lengths = torch.full((4,), -1, dtype=torch.int32, device="cuda")
    ids = torch.zeros(4, T, dtype=torch.long, device="cuda")
    depths = torch.zeros(4, T, dtype=torch.int32, device="cuda")
    visible = torch.zeros(4, T, 1, dtype=torch.int64, device="cuda")
    keep = torch.full((4, T), -1, dtype=torch.int32, device="cuda")
    parents = torch.arange(4, dtype=torch.int32, device="cuda")

    def step():
        cache.fork(lengths, parents, T)
        out = stack.verify(ids, lengths, depths, visible)
        lengths.copy_(stack.accept(lengths, keep))
        return out

    if captured:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()  # all rows idle
        torch.cuda.synchronize()
        assert not bool(cache.refs.any()) and lengths.tolist() == [-1] * 4
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
    prompts()
    lengths.copy_(torch.tensor(lens))
    done = dict.fromkeys(live, 0)
    for _ in range(steps):
        drafts = {}
        for b in live:
            tree = [-1] + [rng.randint(max(0, j - 3), j - 1) for j in range(1, T)]
            depth, on, token = [0], [0], [tail[b][done[b]]]
            for j in range(1, T):
                depth.append(depth[tree[j]] + 1)
                real = tree[j] == on[-1] and rng.random() < 0.7
                token.append(tail[b][done[b] + depth[j]] if real else rng.randrange(512))
                on += [j] if real else []
            drafts[b] = on
            ids[b], depths[b] = torch.tensor(token), torch.tensor(depth)
            visible[b] = kernels.tree_masks(tree)
            keep[b] = torch.tensor(on + [-1] * (T - len(on)))
        keep[1] = 0
        if captured:
            graph.replay()
            logits = out.float()
        else:
            logits = step().float()
        for b, on in drafts.items():
            for d, node in enumerate(on):
                y = want[done[b] + d][b]
                assert float((logits[b, node] - y).norm() / y.norm()) < CLOSE, (b, d)
            done[b] += len(on)
        assert lengths.tolist() == [n + done[b] if n >= 0 else -1 for b, n in enumerate(lens)]
        assert bool((cache.block_table[1] == -1).all())
    kernels.check_device()
    table, refs = cache.block_table, cache.refs
    assert torch.equal(torch.bincount(table[table >= 0].long(), minlength=len(refs)).int(), refs)
    assert max(done.values()) > 16
