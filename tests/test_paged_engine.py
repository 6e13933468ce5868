"""The engine over a paged cache: prompts of different lengths, sampled tokens.

The same 2-layer random-init checkpoint as ``test_engine_gpu`` (head_dim 64).  Numbers are compared
where the model is continuous: the paged stack against the static one with the same stand-in MoE.
Their arithmetic differs by some ten fp16 roundings a layer (the rotation in fp32 instead of fp16,
attention's probabilities, residual sums of slightly different terms), each 2^-11 / sqrt(3) rms of
its value: 20 of them in two layers give 1.3e-3 of relative error; 5e-3 is allowed.  With experts a
router logit within an ulp of the next can pick another expert, so there greedy tokens are compared.
"""
from __future__ import annotations

import pytest
import torch

from tests.test_engine_gpu import KV, L, V, _config, _generate, ckpt  # noqa: F401 (fixture)

gpu = pytest.mark.gpu
PAGED = {"paged_kv": True, "page_size": 16, "max_batch": 3}


def _ragged(lens, seed=1, left=False):
    g = torch.Generator().manual_seed(seed)
    rows = [torch.randint(0, V, (n,), generator=g) for n in lens]
    ids = torch.zeros(len(lens), max(lens), dtype=torch.long)
    mask = torch.zeros_like(ids)
    for b, r in enumerate(rows):
        at = slice(max(lens) - len(r), None) if left else slice(0, len(r))
        ids[b, at], mask[b, at] = r, 1
    return rows, ids, mask


def _run(cfg, ids, mask, n, sampling=None):
    from moeinfra_b200.engine.engine import InferenceEngine
    from moeinfra_b200.engine.types import ForwardRequest

    with InferenceEngine(cfg) as eng:
        return eng.generate(ForwardRequest(ids, mask, n, sampling)), eng


@gpu
@pytest.mark.parametrize("graphs", [True, False])
def test_ragged_prompts_match_single_sequences(ckpt, graphs):  # noqa: F811
    rows, ids, mask = _ragged([12, 1, 33])
    n = 6
    res, _ = _run(_config(ckpt, engine=PAGED | {"cuda_graphs": graphs}), ids, mask, n)
    assert res.stage_timings["cuda_graph_decode"] is graphs
    for b, row in enumerate(rows):
        one, _ = _generate(_config(ckpt), row[None], n)
        assert sum(x == y for x, y in zip(res.token_ids[b], one.token_ids)) >= n - 1


class LinearMoE:
    def __init__(self, w):
        self.w = w

    def forward(self, x):
        return x @ self.w.t()


@gpu
@pytest.mark.parametrize("heads,kv,hd", [(4, 2, 64), (4, 1, 128), (2, 2, 128)])
def test_paged_stack_matches_the_static_one(heads, kv, hd):
    """Prefill of ragged prompts and six decode steps, sequence by sequence in the static stack."""
    from moeinfra_b200.engine.dense import DenseConfig, DenseStack
    from moeinfra_b200.engine.paged import PagedDenseStack
    from moeinfra_b200.model.types import LayerWeights

    hidden, layers, vocab, steps, g = 256, 2, 512, 6, torch.Generator().manual_seed(hd + kv)

    def r(*shape):
        return torch.randn(*shape, generator=g) * 0.05

    weights = [LayerWeights(1 + r(hidden), r(heads * hd, hidden), r(kv * hd, hidden),
                            r(kv * hd, hidden), r(hidden, heads * hd), 1 + r(hidden),
                            torch.zeros(8, hidden)) for _ in range(layers)]
    moes = [LinearMoE(r(hidden, hidden).half().cuda()) for _ in range(layers)]
    cfg = DenseConfig(hidden, heads, kv, hd, vocab, 1e6, 1e-5)
    args = (cfg, weights, r(vocab, hidden), 1 + r(hidden), r(vocab, hidden), moes, "cuda")
    rows, _, _ = _ragged([12, 1, 33, 150])
    tail = torch.randint(0, vocab, (steps, len(rows)), generator=g).cuda()
    with torch.no_grad():
        paged = PagedDenseStack(*args, max_batch=4, max_len=160, page_size=16)
        paged.cache.reserve([len(x) + steps for x in rows])
        got = [paged.prefill(rows)]
        pos = torch.tensor([len(x) for x in rows], dtype=torch.int32, device="cuda")
        for i in range(steps):
            got.append(paged.decode(tail[i][:, None], pos))
            pos += 1
        for b, row in enumerate(rows):
            static = DenseStack(*args, max_batch=1, max_len=160)
            want = [static.forward(row[None].cuda())]
            for i in range(steps):
                at = torch.tensor([len(row) + i], device="cuda")
                want.append(static.forward(tail[i, b].view(1, 1), decode_pos=at))
            for i, (x, y) in enumerate(zip(got, want)):
                x, y = x[b].float(), y[0].float()
                assert float((x - y).norm() / y.norm()) < 5e-3, (b, i)


@gpu
def test_every_batch_of_a_wide_stack_decodes():
    """Batches of 1 to max_batch over tables of 2048 positions, which attention splits otherwise from
    one number of sequences to the next, all with the stack's one workspace."""
    from moeinfra_b200.engine.dense import DenseConfig
    from moeinfra_b200.engine.paged import PagedDenseStack
    from moeinfra_b200.model.types import LayerWeights

    hidden, heads, kv, hd, vocab, g = 256, 32, 8, 64, 512, torch.Generator().manual_seed(9)

    def r(*shape):
        return torch.randn(*shape, generator=g) * 0.05

    weights = [LayerWeights(1 + r(hidden), r(heads * hd, hidden), r(kv * hd, hidden),
                            r(kv * hd, hidden), r(hidden, heads * hd), 1 + r(hidden),
                            torch.zeros(8, hidden))]
    args = (DenseConfig(hidden, heads, kv, hd, vocab, 1e6, 1e-5), weights, r(vocab, hidden),
            1 + r(hidden), r(vocab, hidden), [LinearMoE(r(hidden, hidden).half().cuda())], "cuda")
    rows, _, _ = _ragged([5 + 3 * i for i in range(32)])
    tail = torch.randint(0, vocab, (32, 1), generator=g).cuda()
    with torch.no_grad():
        stack = PagedDenseStack(*args, max_batch=32, max_len=2048, page_size=64)
        want = None
        for B in (32, 19, 18, 8, 1):
            stack.cache.reserve([len(x) + 1 for x in rows[:B]])
            stack.prefill(rows[:B])
            pos = torch.tensor([len(x) for x in rows[:B]], dtype=torch.int32, device="cuda")
            got = stack.decode(tail[:B], pos).float()
            want = got if want is None else want
            err = (got - want[:B]).norm(dim=-1) / want[:B].norm(dim=-1)
            assert float(err.max()) < 5e-3, B


@gpu
def test_padding_side_batch_order_and_graphs_do_not_matter(ckpt):  # noqa: F811
    rows, ids, mask = _ragged([12, 1, 33])
    _, lids, lmask = _ragged([12, 1, 33], left=True)
    a, _ = _run(_config(ckpt, engine=PAGED), ids, mask, 6)
    b, _ = _run(_config(ckpt, engine=PAGED), lids, lmask, 6)
    c, _ = _run(_config(ckpt, engine=PAGED | {"cuda_graphs": False}), ids, mask, 6)
    assert a.token_ids == b.token_ids == c.token_ids
    assert torch.equal(a.logits, b.logits) and torch.equal(a.logits, c.logits)


@gpu
def test_one_engine_serves_requests_in_turn(ckpt):  # noqa: F811
    """Pages return to the pool; a second request's results do not depend on the first."""
    from moeinfra_b200.engine.engine import InferenceEngine
    from moeinfra_b200.engine.types import ForwardRequest

    # 3 + 1 + 2 pages of 16 are needed at most: 6 suffice for either request, not for both.
    cfg = _config(ckpt, engine=PAGED | {"kv_pages": 6})
    first, second = _ragged([33, 3, 20], seed=4), _ragged([5, 40], seed=5)
    with InferenceEngine(cfg) as eng:
        got = [eng.generate(ForwardRequest(ids, mask, 4)) for _, ids, mask in (first, second, first)]
        with pytest.raises(RuntimeError, match="free pages"):
            eng.generate(ForwardRequest(*_ragged([40, 40, 40])[1:], 4))
        again = eng.generate(ForwardRequest(second[1], second[2], 4))
    assert got[0].token_ids == got[2].token_ids and got[1].token_ids == again.token_ids
    alone, _ = _run(cfg, second[1], second[2], 4)
    assert alone.token_ids == again.token_ids


@gpu
def test_offloaded_experts_with_pages(ckpt):  # noqa: F811
    rows, ids, mask = _ragged([7, 19])
    res, _ = _run(_config(ckpt, engine=PAGED), ids, mask, 5)
    off, eng = _run(_config(ckpt, cache={"gpu_slots": 3}, engine=PAGED | {"preload_experts": False}),
                    ids, mask, 5)
    assert off.stage_timings["cuda_graph_decode"] is False and off.token_ids == res.token_ids


@gpu
@pytest.mark.parametrize("paged", [True, False])
def test_sampling(ckpt, paged):  # noqa: F811
    from moeinfra_b200.engine.types import SamplingParams

    over = PAGED if paged else {"max_batch": 3}
    g = torch.Generator().manual_seed(7)
    ids, n = torch.randint(0, V, (3, 10), generator=g), 12
    greedy, _ = _run(_config(ckpt, engine=over), ids, None, n)
    cold, _ = _run(_config(ckpt, engine=over), ids, None, n, SamplingParams(temperature=0.0))
    assert cold.token_ids == greedy.token_ids
    one, _ = _run(_config(ckpt, engine=over), ids, None, n, SamplingParams(top_k=1, seed=1))
    assert one.token_ids == greedy.token_ids
    hot = SamplingParams(temperature=[1.5, 0.0, 0.7], top_k=[0, 0, 20], top_p=[0.95, 1.0, 0.8], seed=3)
    a, _ = _run(_config(ckpt, engine=over), ids, None, n, hot)
    b, _ = _run(_config(ckpt, engine=over), ids, None, n, hot)
    c, _ = _run(_config(ckpt, engine=over | {"cuda_graphs": False}), ids, None, n, hot)
    assert a.token_ids == b.token_ids == c.token_ids
    assert a.token_ids[0] != greedy.token_ids[0]
    hot.seed = 4
    d, _ = _run(_config(ckpt, engine=over), ids, None, n, hot)
    assert d.token_ids[0] != a.token_ids[0]


@gpu
def test_request_checks(ckpt):  # noqa: F811
    from moeinfra_b200.engine.engine import InferenceEngine
    from moeinfra_b200.engine.types import ForwardRequest, SamplingParams

    eng = InferenceEngine(_config(ckpt, engine=PAGED))
    ids = torch.zeros(2, 4, dtype=torch.long)
    empty = torch.tensor([[1, 1, 0, 0], [0, 0, 0, 0]])
    for bad in (ForwardRequest(torch.zeros(4, 4, dtype=torch.long)), ForwardRequest(ids[0]),
                ForwardRequest(ids, empty), ForwardRequest(ids, empty[:1]),
                ForwardRequest(torch.zeros(1, 60, dtype=torch.long), None, 10),
                ForwardRequest(ids, None, -1), ForwardRequest(ids[:, :0]),
                ForwardRequest(ids, None, 2, SamplingParams(top_p=[0.5])),
                ForwardRequest(ids, None, 2, SamplingParams(temperature=-1.0))):
        with pytest.raises(ValueError):
            eng.generate(bad)
    assert len(eng.generate(ForwardRequest(ids, None, 2)).token_ids) == 2
    assert eng.generate(ForwardRequest(ids[:1], None, 0)).token_ids == []
    eng.close()
    with pytest.raises(ValueError, match="multiple of 16"):
        InferenceEngine(_config(ckpt, engine=PAGED | {"page_size": 24})).generate(
            ForwardRequest(ids, None, 2))
    with pytest.raises(ValueError, match="expert_parallel"):
        InferenceEngine(_config(ckpt, engine=PAGED) | {"parallel": {"expert_parallel": True}})


@gpu
@pytest.mark.parametrize("paged", [True, False])
@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("sampled", [True, False])
def test_decoding_waits_for_the_device_once(ckpt, paged, graphs, sampled):  # noqa: F811
    """The tokens' way back is the only point where the host waits in the decode stage."""
    import warnings

    from moeinfra_b200.engine.engine import InferenceEngine, _Sampler
    from moeinfra_b200.engine.types import ForwardRequest, SamplingParams

    over = (PAGED if paged else {"max_batch": 3}) | {"cuda_graphs": graphs}
    ids = torch.randint(0, V, (3, 10), generator=torch.Generator().manual_seed(7))
    params = SamplingParams(seed=1) if sampled else None
    with InferenceEngine(_config(ckpt, engine=over)) as eng:
        want = eng.generate(ForwardRequest(ids, None, 6, params)).token_ids
        logits = eng._prefill(ids)
        sampler = _Sampler(params, 3, 6, eng._device) if sampled else None
        torch.cuda.synchronize()
        torch.cuda.set_sync_debug_mode("warn")
        try:
            with warnings.catch_warnings(record=True) as seen:
                warnings.simplefilter("always")
                got = eng._decode(logits, 6, sampler)
        finally:
            torch.cuda.set_sync_debug_mode("default")
        assert got == want
        assert sum("synchronizing" in str(w.message) for w in seen) == 1, [str(w) for w in seen]


def test_cache_hands_out_and_takes_back_pages():
    """Host logic of the page pool (CPU)."""
    from moeinfra_b200.engine.paged import PagedKVCache

    c = PagedKVCache(1, 5, 1, 16, 64, max_batch=3, max_len=64, device="cpu")
    assert c.block_table.shape == (3, 4) and c.free_pages == 5
    c.reserve([17, 0, 33])
    held = c.block_table[c.block_table >= 0].tolist()
    assert sorted(held) == [0, 1, 2, 3, 4] and c.free_pages == 0
    assert (c.block_table >= 0).sum(1).tolist() == [2, 0, 3]
    c.reserve([64])  # what was held before comes back first
    assert c.free_pages == 1 and (c.block_table >= 0).sum().item() == 4
    with pytest.raises(RuntimeError, match="free pages"):
        c.reserve([64, 32])
    with pytest.raises(ValueError):
        c.reserve([65])
    with pytest.raises(ValueError):
        c.reserve([1] * 4)
    c.release()
    c.release()
    assert c.free_pages == 5
    with pytest.raises(ValueError):
        PagedKVCache(1, 5, 1, 8, 64, 3, 64, "cpu")
