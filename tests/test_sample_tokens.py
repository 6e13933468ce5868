"""The sampler against its definition in Python integers, and against a sort on the GPU.

Tokens are whole numbers and have to be equal wherever the definition's own exponential leaves no
doubt (``oracle.serving.sample``); against torch on the same GPU, whose exponential is the same
function, they have to be equal everywhere.  A probability is one division of two such sums: half a
unit in fp32's last place, and 2^-21 of it for the exponentials.
"""
from __future__ import annotations

import pytest
import torch

from oracle import serving as ref

gpu = pytest.mark.gpu
SCALE = float(1 << 40)


def _params(rows, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    def full(v, dtype):
        return torch.tensor(v if isinstance(v, list) else [v] * rows, dtype=dtype, device="cuda")

    return (full(temperature, torch.float32), full(top_k, torch.int32),
            full(top_p, torch.float32), full(min_p, torch.float32))


def _sorted_form(x, u, temperature, top_k, top_p, min_p):
    """The definition with a sort, in torch on the GPU (int64 sums)."""
    x = x.float() + 0.0
    V = x.shape[1]
    x = x.masked_fill(x.isnan(), float("-inf"))
    greedy = (temperature <= 0)[:, None]
    T = temperature[:, None].masked_fill(greedy, 1.0)
    k = top_k[:, None].long()
    k = torch.where(greedy, 1, torch.where(k > 0, k, V))
    top = x.amax(-1, keepdim=True)
    e = torch.exp(torch.where(x == top, 0.0, (x - top) / T))
    w = (e * SCALE).long()
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    ws, es = w.gather(1, order), e.gather(1, order)
    keep = torch.arange(V, device=x.device)[None] < k
    cum = (ws * keep).cumsum(-1)
    total = cum[:, -1:]
    p = top_p[:, None]
    need = torch.where(p < 1, torch.ceil(p.double() * total.double()).long(), total)
    keep &= cum - ws < need.clamp(min=1)
    keep &= es >= min_p[:, None].clamp(max=1.0)
    kept = torch.zeros_like(w).scatter_(1, order, ws * keep)
    cum = kept.cumsum(-1)
    total = cum[:, -1:]
    r = torch.floor(u[:, None].double() * total.double()).long().clamp(min=0)
    tokens = (cum > torch.minimum(r, total - 1)).long().argmax(-1)
    return tokens, (kept.gather(1, tokens[:, None]).double() / total.double())[:, 0].float()


def _compare(x, u, params):
    from moeinfra_b200 import kernels

    tokens, probs = kernels.sample_tokens(x, u, *params)
    want, want_p = _sorted_form(x, u, *params)
    assert torch.equal(tokens, want)
    torch.testing.assert_close(probs, want_p, rtol=2.0 ** -22, atol=0)
    return tokens, probs


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 63, 1000, 1003])
def test_against_integers(dtype, vocab):
    from moeinfra_b200 import kernels

    g = torch.Generator().manual_seed(vocab)
    cases = [(t, k, p, m) for t in (0.0, 0.5, 1.0, 3.0) for k in (0, 1, 2, 40)
             for p in (1.0, 0.9, 0.3, 0.0) for m in (0.0, 0.1, 1.0)]
    rows = len(cases)
    x = (3 * torch.randn(rows, vocab, generator=g)).to(dtype)
    u = torch.rand(rows, generator=g)
    u[::7], u[3::7] = 0.0, 1 - 2.0 ** -24
    t, k, p, m = (list(v) for v in zip(*cases))
    tokens, probs = kernels.sample_tokens(x.cuda(), u.cuda(), *_params(rows, t, k, p, m))
    unsure = 0
    for i in range(rows):
        token, prob, sure = ref.sample(x[i].float().numpy(), float(u[i]), *cases[i])
        if not sure:
            unsure += 1
            continue
        assert int(tokens[i]) == token, cases[i]
        assert abs(float(probs[i]) - prob) <= (2.0 ** -24 + 2.0 ** -21) * prob
    # u = 0 or nearly 1 with a single token kept, p = 0 and ties leave no margin in a few rows.
    assert unsure < rows


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(1, 32000), (3, 4095), (3, 4097), (64, 32000), (5, 50001),
                                        (300, 5000), (2, 131072), (1, 131073), (2, 262144)])
def test_against_a_sort(dtype, rows, vocab):
    """Every split of a row over CTAs and threads, mixed parameters."""
    g = torch.Generator(device="cuda").manual_seed(rows + vocab)
    x = 2.5 * torch.randn(rows, vocab, device="cuda", generator=g)
    x += (torch.rand(rows, vocab, device="cuda", generator=g) < 100 / vocab) * 6.0
    u = torch.rand(rows, device="cuda", generator=g)

    def cycle(values):
        return [values[i % len(values)] for i in range(rows)]

    for shift in range(3):
        params = _params(rows, cycle([0.8, 1.0, 0.0, 1.7, 0.2][shift:]),
                         cycle([0, 50, 0, 1, 1000, vocab][shift:]),
                         cycle([0.95, 1.0, 0.5, 0.99][shift:]), cycle([0.0, 0.0, 0.05][shift:]))
        _compare(x.to(dtype), u, params)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_ties_go_to_the_lowest_index(dtype):
    """Few distinct logits: every boundary falls among equal ones."""
    g = torch.Generator(device="cuda").manual_seed(1)
    rows, vocab = 60, 20000
    x = torch.randint(0, 4, (rows, vocab), device="cuda", generator=g).to(dtype)
    u = torch.rand(rows, device="cuda", generator=g)
    cyc = [(0, 0.5), (7, 1.0), (6000, 0.9), (0, 1.0), (3, 0.2), (19999, 0.999)] * 10
    _compare(x, u, _params(rows, 1.0, [k for k, _ in cyc], [p for _, p in cyc]))
    flat = torch.zeros(rows, vocab, device="cuda", dtype=dtype)
    tokens, probs = _compare(flat, u, _params(rows, 1.0, [k for k, _ in cyc], [p for _, p in cyc]))
    assert all(int(t) < 7 for t, (k, p) in zip(tokens, cyc) if k == 7)
    zeros = torch.zeros(2, 9, device="cuda", dtype=dtype)
    zeros[:, 4:] = -0.0
    _compare(zeros, u[:2], _params(2, 1.0, 5, 1.0))  # -0 and 0 are equal


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_infinities_nan_and_extremes(dtype):
    inf, nan = float("inf"), float("nan")
    big = torch.finfo(dtype).max
    rows = [[-inf, 1.0, 2.0, -inf], [nan, 1.0, 0.0, nan], [-inf] * 4, [nan] * 4,
            [inf, 1.0, inf, -inf], [-big, -big, big, 0.0], [-big] * 4, [0.0, -big, nan, -inf]]
    x = torch.tensor(rows, device="cuda").to(dtype).repeat(8, 1)
    u = (torch.arange(64, device="cuda") + 0.5) / 64
    for kw in (dict(), dict(top_k=2), dict(top_p=0.6), dict(min_p=0.3), dict(temperature=0.0),
               dict(temperature=1e-6), dict(temperature=1e6, top_k=3, top_p=0.8), dict(temperature=3e38),
               dict(temperature=1e-38), dict(temperature=1e-45, top_p=0.9)):
        tokens, _ = _compare(x, u, _params(64, **kw))
        for i, t in enumerate(tokens.tolist()):  # a masked token is drawn only where all are
            row = rows[i % 8]
            if any(v > -inf for v in row):
                assert row[t] > -inf


@gpu
def test_odd_numbers():
    """Random numbers and parameters outside their ranges: some kept token, no fault."""
    from moeinfra_b200 import kernels

    x = torch.tensor([[0.0, 3.0, 1.0]], device="cuda").repeat(7, 1)
    u = torch.tensor([-1.0, 1.0, 2.0, float("nan"), float("inf"), 0.5, 0.5], device="cuda")
    nan = float("nan")
    tokens, probs = kernels.sample_tokens(
        x, u, *_params(7, [1, 1, 1, 1, 1, nan, -1.0], [0, 0, -3, 9, 0, 0, 0],
                       [1, 2.0, -1.0, 1, nan, 1, 1], [0, 0, 0, 0, 0, 0, 5.0]))
    assert tokens.tolist() == [0, 2, 1, 0, 2, 1, 1]
    assert (probs > 0).all() and (probs <= 1).all()


@gpu
def test_strides_streams_and_batches_do_not_matter():
    from moeinfra_b200 import kernels

    g = torch.Generator(device="cuda").manual_seed(5)
    rows, vocab = 90, 9001  # rows not 16-byte aligned
    wide = 3 * torch.randn(rows, vocab + 6, device="cuda", generator=g).half()
    x = wide[:, 3:3 + vocab]
    u = torch.rand(rows, device="cuda", generator=g)
    params = _params(rows, 0.9, 200, 0.9)
    tokens, probs = _compare(x, u, params)
    packed = kernels.sample_tokens(x.contiguous(), u, *params)
    assert torch.equal(packed[0], tokens) and torch.equal(packed[1], probs)
    for i in (0, 41, 89):  # alone, a row is split otherwise
        one = kernels.sample_tokens(x[i:i + 1], u[i:i + 1], *(p[i:i + 1] for p in params))
        assert int(one[0]) == int(tokens[i]) and float(one[1]) == float(probs[i])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = kernels.sample_tokens(x, u, *params)
    s.synchronize()
    assert torch.equal(other[0], tokens)
    assert kernels.sample_tokens(x[:0], u[:0], *(p[:0] for p in params))[0].shape == (0,)


@gpu
def test_frequencies_follow_the_probabilities():
    """4096 evenly spread numbers hit each kept token as often as its probability says, to 1."""
    from moeinfra_b200 import kernels

    n = 4096
    x = torch.tensor([1.0, -2.0, 3.0, 2.5, 0.0, 2.9], device="cuda").repeat(n, 1)
    u = (torch.arange(n, device="cuda") + 0.5) / n
    tokens, probs = kernels.sample_tokens(x, u, *_params(n, 0.7, 4, 0.98))
    e, order = torch.softmax(x[0].double() / 0.7, 0).sort(descending=True)
    e, order = e[:4], order[:4]
    n_kept = int((e.cumsum(0) < 0.98 * e.sum()).sum()) + 1
    kept, share = order[:n_kept].tolist(), e[:n_kept] / e[:n_kept].sum()
    assert sorted(set(tokens.tolist())) == sorted(kept)
    for i, s in zip(kept, share.tolist()):
        assert abs(int((tokens == i).sum()) - s * n) <= 1
        assert abs(float(probs[tokens == i][0]) - s) < 1e-6


def test_host_checks_precede_every_launch():
    from moeinfra_b200 import _native

    lib, f = _native.lib(), 0x100000

    def sample(logits=f, stride=100, rows=3, vocab=100, dtype=0, u=f, out=f):
        return lib.moe_sample_tokens(_native.SAMPLE_TOKENS.pack(
            logits, stride, rows, vocab, dtype, u, f, f, f, f, out, f, 0))

    assert sample(rows=0) == 0 and lib.moe_sample_tokens(None) == 1
    assert sample(rows=-1) == 1 and sample(vocab=0) == 1 and sample(stride=99) == 1
    assert sample(logits=0) == 1 and sample(u=0) == 1 and sample(out=0) == 1
    assert sample(dtype=3) == 2 and sample(vocab=262145, stride=262145) == 2


def test_wrapper_refuses_cpu_tensors():
    from moeinfra_b200 import kernels

    one = torch.ones(1)
    with pytest.raises(RuntimeError, match="no CPU path"):
        kernels.sample_tokens(torch.zeros(1, 8), one, one, one.int(), one, one)


@gpu
def test_wrapper_refuses_wrong_shapes_and_types():
    from moeinfra_b200 import kernels

    x, one = torch.zeros(2, 8, device="cuda"), torch.ones(2, device="cuda")

    def sample(x=x, u=one, t=one, k=one.int(), p=one, m=one):
        return kernels.sample_tokens(x, u, t, k, p, m)

    sample()
    for bad in (dict(x=x.double()), dict(x=x[0]), dict(u=one[:1]), dict(k=one), dict(t=one.half()),
                dict(p=one.double()), dict(m=one[:1]), dict(x=x.t()), dict(u=one[:, None])):
        with pytest.raises(ValueError):
            sample(**bad)


# Long rows, few of them and many: a row over several CTAs, and in one.
@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(6, 20001), (40, 20001), (3, 70000), (40, 70000)])
def test_long_rows_of_few_values(dtype, rows, vocab):
    """Boundaries among thousands of equal logits, and of nearly equal ones."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    steps = torch.randint(0, 5, (rows, vocab), device="cuda", generator=g).float()
    near = 4.0 + 1e-3 * torch.rand(rows, vocab, device="cuda", generator=g)
    u = torch.rand(rows, device="cuda", generator=g)
    for x in (steps.to(dtype), near.to(dtype), torch.zeros_like(steps).to(dtype)):
        for kw in (dict(), dict(top_k=37), dict(top_p=0.7), dict(top_k=5000, top_p=0.31),
                   dict(top_k=vocab - 1, top_p=0.999, min_p=0.2), dict(temperature=0.0)):
            _compare(x, u, _params(rows, **kw))


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [6, 60])
def test_long_rows_of_infinities_and_nan(dtype, rows):
    inf, nan = float("inf"), float("nan")
    big = torch.finfo(dtype).max
    heads = [[-inf, 1.0, 2.0, -inf], [nan, 1.0, 0.0, nan], [-inf] * 4, [inf, 1.0, inf, -inf],
             [-big, -big, big, 0.0], [-big] * 4]
    x = torch.full((rows, 20000), -inf, device="cuda")
    x[:, 1::3] = nan
    x[:, 9998:10002] = torch.tensor(heads, device="cuda").repeat(rows // 6, 1)
    x = x.to(dtype)
    u = (torch.arange(rows, device="cuda") + 0.5) / rows
    for kw in (dict(), dict(top_k=2), dict(top_p=0.6), dict(min_p=0.3), dict(temperature=0.0),
               dict(temperature=1e6, top_k=3, top_p=0.8), dict(temperature=3e38),
               dict(temperature=1e-38), dict(temperature=1e-45, top_p=0.9)):
        tokens, _ = _compare(x, u, _params(rows, **kw))
        assert tokens.min() >= 0 and tokens.max() < 20000


@gpu
@pytest.mark.parametrize("top_k,top_p,min_p", [(0, 0.999, 0.0), (3000, 1.0, 0.0), (20000, 0.98, 0.0),
                                               (0, 0.99, 1e-3), (300, 0.5, 0.0), (0, 0.01, 0.0)])
def test_many_kept(top_k, top_p, min_p):
    """More candidates than the lists hold, just as many, and few, in one call."""
    g = torch.Generator(device="cuda").manual_seed(11)
    rows, vocab = 60, 50000
    x = torch.randn(rows, vocab, device="cuda", generator=g)
    x *= torch.linspace(0.05, 6.0, rows, device="cuda")[:, None]
    u = torch.rand(rows, device="cuda", generator=g)
    _compare(x, u, _params(rows, 1.0, top_k, top_p, min_p))


# Rows over several CTAs with top-k and top-p together: the boundary of the second lies among the
# logits that the first one's search gathered last.
@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(1, 32000), (7, 32000), (2, 131072), (10, 131072)])
def test_top_p_near_the_cut_of_top_k(dtype, rows, vocab):
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = 2 * torch.randn(rows, vocab, device="cuda", generator=g)
    x += (torch.rand(rows, vocab, device="cuda", generator=g) < 200 / vocab) * (
        3 + 2.5 * torch.randn(rows, vocab, device="cuda", generator=g).abs())
    u = torch.rand(rows, device="cuda", generator=g)
    for t in (0.7, 1.0, 2.0):
        for k in (1000, 2000, 5000, 10000, 20000):
            for p in (0.9, 0.99, 0.999):
                _compare(x.to(dtype), u, _params(rows, t, k, p))


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(1, 32000), (5, 32000), (3, 131072), (1, 200000)])
def test_top_p_near_the_cut_of_top_k_among_ties(dtype, rows, vocab):
    """Thousands of logits equal to the cut, so that every search's lists are full of them."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    flat = torch.zeros(rows, vocab, device="cuda")
    flat[:, 100:105] = 3.0
    few = torch.randint(0, 3, (rows, vocab), device="cuda", generator=g) * 1e-3
    few[:, ::7] = few[:, ::7] + 2 ** -9
    u = torch.rand(rows, device="cuda", generator=g)
    for x in (flat, few):
        for k in (1000, 10000, 20000, vocab - 1):
            for p in (0.5, 0.99, 0.9999):
                _compare(x.to(dtype), u, _params(rows, 1.0, k, p))


@gpu
def test_a_wait_that_runs_out_ends_the_call():
    """With no time to wait, a row's CTAs give up at different points: the call ends with a status at
    most, and the next one is right."""
    from moeinfra_b200 import _native, kernels

    g = torch.Generator(device="cuda").manual_seed(2)
    rows, vocab = 30, 131072
    x = torch.randn(rows, vocab, device="cuda", generator=g).half()
    u = torch.rand(rows, device="cuda", generator=g)
    kinds = [dict(temperature=0.0), dict(), dict(top_p=0.9), dict(top_k=5000, top_p=0.99),
             dict(temperature=0.1, top_k=20)]
    old = _native.wait_limit_ns()
    for kw in kinds:
        params = _params(rows, **kw)
        _native.set_wait_limit_ns(1000)
        try:
            for _ in range(20):
                kernels.sample_tokens(x, u, *params)
            try:
                kernels.check_device()
            except RuntimeError as e:
                assert "timed out" in str(e)
        finally:
            _native.set_wait_limit_ns(old)
        _compare(x, u, params)
        kernels.check_device()


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_lists_that_fill_while_they_are_gathered(dtype):
    """From just under to just over the 2048 logits a list holds, row by row: warps meet a list that
    others have filled in between."""
    g = torch.Generator(device="cuda").manual_seed(3)
    rows, vocab = 150, 40000
    x = torch.randn(rows, vocab, device="cuda", generator=g).to(dtype)
    u = torch.rand(rows, device="cuda", generator=g)
    k = [1800 + 5 * i for i in range(rows)]
    for kw in (dict(top_k=k), dict(top_k=k, min_p=0.05), dict(top_k=k, top_p=0.9),
               dict(top_p=[0.05 + 0.003 * i for i in range(rows)])):
        _compare(x, u, _params(rows, 0.7, **kw))


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [20001, 70001, 140001])
def test_a_row_alone_and_in_a_batch(dtype, vocab):
    """40 rows take a CTA each, one row is spread over a cluster (8, 16 or 32 logits a thread): the
    same token and the same bits of its probability."""
    from moeinfra_b200 import kernels

    g = torch.Generator(device="cuda").manual_seed(vocab)
    rows = 40
    x = 2.5 * torch.randn(rows, vocab, device="cuda", generator=g)
    x[::5] = x[::5].round()  # thousands of ties
    x[::7, ::3] = float("nan")
    x = x.to(dtype)
    u = torch.rand(rows, device="cuda", generator=g)

    def cycle(values):
        return [values[i % len(values)] for i in range(rows)]

    for shift in range(2):
        params = _params(rows, cycle([0.8, 1.0, 0.0, 1.7][shift:]), cycle([0, 50, 3000, 0, 1, 1000][shift:]),
                         cycle([0.95, 1.0, 0.999, 0.5][shift:]), cycle([0.0, 0.0, 0.05][shift:]))
        tokens, probs = _compare(x, u, params)
        for i in range(rows):
            token, prob = kernels.sample_tokens(x[i:i + 1], u[i:i + 1], *(p[i:i + 1] for p in params))
            assert torch.equal(token[0], tokens[i]) and torch.equal(prob[0], probs[i]), i


@gpu
@pytest.mark.parametrize("rows,vocab", [(5, 20001), (200, 3000)])
def test_several_tokens_of_one_row(rows, vocab):
    """A row expanded, not copied: as many draws as random numbers."""
    g = torch.Generator(device="cuda").manual_seed(6)
    x = 3 * torch.randn(1, vocab, device="cuda", generator=g).half()
    u = torch.rand(rows, device="cuda", generator=g)
    tokens, _ = _compare(x.expand(rows, vocab), u, _params(rows, 1.0, 0, 0.95))
    assert len(set(tokens.tolist())) > 1
