"""beam_select against the definition in 64 bits.

How far a score may be off: the exponentials (2^-22 each, their arguments' rounding less than that
where a term counts), the sums (three steps in fp32, then fp64) and the parts' factors leave the sum
within 2^-20, so its logarithm too; the logarithm, the two differences and the result are rounded
once each, by 2^-24 of their sizes.  A token may stand in another's place only where their exact
scores are nearer than twice that.
"""
from __future__ import annotations

import math

import pytest
import torch

from oracle import branches

gpu = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def _off(v, score):
    """The bound at a score v of a beam with running score `score`: |d - ln sum| <= |v - score| and
    ln sum <= 14 (vocab <= 2^20)."""
    return 2.0 ** -20 + 2.0 ** -24 * (14 + abs(v - score) + abs(v))


def _check(logits, scores, count, got):
    groups, K = scores.shape
    got = [t.cpu() for t in got]
    for t, dt in zip(got, (torch.float32, torch.int32, torch.int64)):
        assert t.shape == (groups, count) and t.dtype == dt
    for b in range(groups):
        x = logits[b * K:(b + 1) * K].cpu()
        want, parents, tokens = branches.beam_select(x, scores[b].cpu(), count)
        xd = x.double()
        xd = torch.where(xd.isnan(), -math.inf, xd)
        d = torch.where(xd == xd.amax(-1, keepdim=True), 0.0, xd - xd.amax(-1, keepdim=True))
        lse = d.exp().sum(-1).log()
        seen = set()
        for j in range(count):
            v, p, t = float(got[0][b, j]), int(got[1][b, j]), int(got[2][b, j])
            if want[j] == -math.inf:
                assert (v, p, t) == (-math.inf, 0, 0)
                continue
            exact = float(scores[b, p]) + float(d[p, t] - lse[p])
            off = _off(exact, float(scores[b, p]))
            assert abs(v - exact) <= off, (b, j, v, exact)
            if (p, t) != (parents[j], tokens[j]):
                assert abs(exact - float(want[j])) <= 2 * off, (b, j, exact, float(want[j]))
            seen.add((p, t))
        assert len(seen) == int((want > -math.inf).sum())


def _logits(rows, vocab, dtype, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = spread * torch.randn(rows, vocab, generator=g)
    x += (torch.rand(rows, vocab, generator=g) < 50 / vocab) * 6.0
    return x.to(dtype).cuda()


def _scores(groups, beams, seed):
    g = torch.Generator().manual_seed(seed + 1)
    return (-20 + 3 * torch.randn(groups, beams, generator=g)).cuda()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("groups,beams,vocab,count", [
    (1, 1, 1, 1), (1, 1, 1, 3), (3, 2, 5, 4), (2, 4, 100, 64), (1, 4, 32000, 4), (5, 3, 32001, 6),
    (16, 4, 31999, 8), (1, 1, 131073, 2), (2, 64, 4097, 64), (40, 16, 1031, 32), (1, 8, 262147, 16)])
def test_against_64_bits(groups, beams, vocab, count, dtype):
    from moeinfra_b200 import kernels

    x, s = _logits(groups * beams, vocab, dtype, vocab), _scores(groups, beams, vocab)
    got = kernels.beam_select(x, s, count)
    kernels.check_device()
    _check(x, s, count, got)
    again = kernels.beam_select(x, s, count)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shift,pad", [(1, 3), (3, 0), (5, 8)])
def test_strided_rows_at_any_element(dtype, shift, pad):
    from moeinfra_b200 import kernels

    rows, vocab = 6, 1003
    buf = torch.full((rows, shift + vocab + pad), 50.0, dtype=dtype, device="cuda")
    buf[:, shift:shift + vocab] = _logits(rows, vocab, dtype, 3)
    s = _scores(2, 3, 3)
    got = kernels.beam_select(buf[:, shift:shift + vocab], s, 5)
    _check(buf[:, shift:shift + vocab], s, 5, got)
    one = buf[:1, shift:shift + vocab].expand(rows, vocab)
    _check(one, s, 5, kernels.beam_select(one, s, 5))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count", [1, 8, 64])
def test_equal_and_sorted_logits(dtype, count):
    """Rows of one value, of few values, rising and falling: the list overflows and is searched in
    rounds; equal scores go to the lower beam, then the lower token (all is exact here)."""
    from moeinfra_b200 import kernels

    vocab = 70001
    ramp = torch.arange(vocab, dtype=torch.float32)
    rows = torch.stack([torch.full((vocab,), 2.0), (ramp % 3), ramp / vocab * 8, -ramp / vocab * 8,
                        torch.where(ramp == 69998, 1.0, 0.0), (ramp % 1000 == 999) * 4.0])
    x = rows.to(dtype).cuda()
    for k in range(6):
        one = x[k:k + 1].contiguous()
        s = torch.zeros(1, 1, device="cuda")
        got = kernels.beam_select(one, s, count)
        want = torch.sort(one[0].cpu(), descending=True, stable=True).indices[:count]
        assert torch.equal(got[2][0].cpu(), want), k
        _check(one, s, count, got)
    twin = x[:1].expand(4, vocab)
    got = kernels.beam_select(twin, torch.tensor([[-1.0, -1.0], [-2.0, -1.0]], device="cuda"), count)
    assert got[2].tolist() == [list(range(count))] * 2
    assert got[1].tolist() == [[0] * count, [1] * count]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count", [1, 16, 64])
def test_long_stretches_of_sorted_and_tied_logits(dtype, count):
    """As many rows as leave each to one CTA, so that its stretches grow: rising (every stretch
    overflows), falling, noise of few values (ties at the threshold) and of many, a late plateau."""
    from moeinfra_b200 import kernels

    vocab, rows = 70001, 600
    ramp = torch.arange(vocab, dtype=torch.float32)
    noise = torch.randn(vocab, generator=torch.Generator().manual_seed(5))
    x = torch.stack([ramp / 8192, -ramp / 8192, noise.mul(2).round(), noise, noise + ramp / 65536,
                     torch.where(ramp < 30000, noise, 5.0),
                     torch.where((ramp > 9000) & (ramp < 9000 + count), 7.0, noise.clamp(max=3))])
    x = x.to(dtype).cuda()
    for k in range(len(x)):
        got = kernels.beam_select(x[k:k + 1].expand(rows, vocab), torch.zeros(rows, 1, device="cuda"), count)
        want = torch.sort(x[k].cpu(), descending=True, stable=True).indices[:count]
        assert torch.equal(got[2].cpu(), want.expand(rows, count)), k
        assert not bool(got[1].any()) and bool((got[0] == got[0][:1]).all())
    kernels.check_device()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_and_nan(dtype):
    from moeinfra_b200 import kernels

    inf, nan = math.inf, math.nan
    x = _logits(12, 2050, dtype, 5)
    x[0, ::2] = nan
    x[1] = -inf
    x[2] = nan
    x[3, [7, 1999]] = inf
    x[4] = -inf
    x[4, 77] = -3.0          # an ended beam: its end token alone, log-probability 0
    x[5, :2000] = -inf
    x[6, 2049] = inf
    x[6, 0] = nan
    s = _scores(4, 3, 5)
    s[3] = torch.tensor([-inf, nan, -5.0])
    got = kernels.beam_select(x, s, 7)
    kernels.check_device()
    s = torch.where(s.isnan(), -inf, s)  # the oracle's: a NaN score offers nothing
    _check(x, s, 7, got)
    got = kernels.beam_select(x, s, 64)  # group 1 has 2 + 1 + 50 candidates: all of them
    _check(x, s, 64, got)
    ended = (got[2][1] == 77) & (got[1][1] == 1)
    assert got[0][1][ended].tolist() == [float(s[1, 1])]
    _check(x[1:3], s[:1, :2], 3, kernels.beam_select(x[1:3], s[:1, :2].contiguous(), 3))


@gpu
def test_first_step_and_many_groups():
    """One live beam per group; more groups than a launch has counters."""
    from moeinfra_b200 import kernels

    groups = 2300
    x = _logits(groups * 2, 61, torch.float32, 8)
    s = torch.tensor([[0.0, -math.inf]], device="cuda").repeat(groups, 1)
    got = kernels.beam_select(x, s)
    want = torch.log_softmax(x[::2].double(), -1).topk(2)
    assert torch.equal(got[2], want.indices) and not bool(got[1].any())
    assert float((got[0].double() - want.values).abs().max()) <= _off(20.0, 0.0)
    _check(x[:8], s[:4], 2, [t[:4] for t in got])


@gpu
def test_large_scores_keep_the_logits_order():
    """Far below zero a score's rounding step holds many logits: they stay in the logits' order."""
    from moeinfra_b200 import kernels

    x = torch.linspace(0, 1, 40000, dtype=torch.float32).flip(0)[None].repeat(2, 1).cuda()
    s = torch.tensor([[-1e6, -1e6]], device="cuda")
    got = kernels.beam_select(x, s, 6)
    assert got[2].tolist() == [list(range(6))] and got[1].tolist() == [[0] * 6]
    assert len(set(got[0][0].tolist())) == 1


@gpu
def test_graphs_side_by_side_and_own_workspace():
    from moeinfra_b200 import kernels

    cases = [(_logits(8, 32000, torch.float16, i), _scores(2, 4, i)) for i in range(2)]
    want = [kernels.beam_select(x, s, 8) for x, s in cases]
    graphs, outs = [], []
    for i, (x, s) in enumerate(cases):
        ws = kernels.beam_select_workspace(x, 4, 8) if i else None
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(kernels.beam_select(x, s, 8, workspace=ws))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for a, b in zip(want, outs):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    none = kernels.beam_select(cases[0][0][:0], cases[0][1][:0], 3)
    assert [t.shape for t in none] == [(0, 3)] * 3


def test_refusals_on_the_host():
    from moeinfra_b200 import _native, kernels

    x, s = torch.zeros(4, 10), torch.zeros(2, 2)
    with pytest.raises(RuntimeError, match="no CPU path"):
        kernels.beam_select(x, s)
    with pytest.raises(ValueError, match="logits must be"):
        kernels.beam_select(x[0], s)
    with pytest.raises(ValueError, match="float16, bfloat16 or float32"):
        kernels.beam_select(x.double(), s)
    with pytest.raises(ValueError, match="scores must be"):
        kernels.beam_select(x, s[0])
    lib, fake = _native.lib(), 0x100000

    def call(logits=fake, stride=100, groups=2, beams=2, vocab=100, dt=2, scores=fake, count=2, out=fake,
             ws=fake, nbytes=1 << 20):
        return lib.moe_beam_select(_native.BEAM_SELECT.pack(
            logits, stride, groups, beams, vocab, dt, scores, count, out, fake, fake, ws, nbytes, 0))

    assert lib.moe_beam_select(None) == 1
    assert call(groups=-1) == 1 and call(beams=0) == 1 and call(count=0) == 1 and call(vocab=0) == 1
    assert call(stride=99) == 1 and call(stride=-1) == 1 and call(logits=0) == 1 and call(out=0) == 1
    assert call(beams=65) == 2 and call(count=65) == 2 and call(vocab=(1 << 20) + 1, stride=1 << 21) == 2
    assert call(dt=3) == 2 and call(groups=1 << 40) == 2 and call(groups=0) == 0
    assert call(logits=fake + 2) == 5 and call(ws=fake + 8) == 5 and call(nbytes=4000) == 4
    assert lib.moe_beam_select_workspace_size(2, 65, 100, 2, 2) == 0


@gpu
def test_refusals_by_name():
    from moeinfra_b200 import kernels

    x, s = torch.zeros(4, 10, device="cuda"), torch.zeros(2, 2, device="cuda")
    for args, name in (((x, s.half()), "scores"), ((x, s.cpu()), "scores"), ((x[:3], s), "3 rows"),
                       ((x, s, 65), "1 to 64"), ((x, s, 0), "1 to 64"), ((x.t(), s), "logits"),
                       ((x, s.t()), "scores")):
        with pytest.raises((ValueError, RuntimeError), match=name):
            kernels.beam_select(*args)
    with pytest.raises(ValueError, match="workspace"):
        kernels.beam_select(x, s, workspace=s)


def test_workspace_sizes_rise_with_the_rows():
    """A buffer made for the largest batch serves the smaller ones, of whatever vocabulary and type."""
    from moeinfra_b200 import _native

    size = _native.lib().moe_beam_select_workspace_size
    for count in (1, 8, 64):
        for beams in (1, 4, 64):
            for vocab, dtype in ((1, 0), (32000, 0), (131072, 0), (131072, 2), (1 << 20, 1)):
                sizes = [size(groups, beams, vocab, count, dtype) for groups in range(0, 1300, 1)]
                assert all(a <= b for a, b in zip(sizes, sizes[1:])), (count, beams, vocab, dtype)
                assert sizes[700] >= size(40, beams, 131072, count, 0)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_a_workspace_for_the_largest_batch_serves_every_smaller_one(dtype):
    from moeinfra_b200 import kernels

    vocab, count = 65536, 8
    x, s = _logits(149, vocab, dtype, 3), _scores(149, 1, 3)
    ws = kernels.beam_select_workspace(x, 1, count)
    for rows in (149, 148, 128, 75, 37, 4, 1):
        got = kernels.beam_select(x[:rows], s[:rows], count, workspace=ws)
        want = kernels.beam_select(x[:rows], s[:rows], count)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), rows
    kernels.check_device()
    _check(x[:4], s[:4], count, [t[:4] for t in kernels.beam_select(x, s, count, workspace=ws)])


def _in_place(x, scores, out, beams, count, groups):
    """The library's call with its new scores at ``out``; status, parents, tokens."""
    from moeinfra_b200 import _native, kernels

    parents = torch.zeros(groups, count, dtype=torch.int32, device=x.device)
    tokens = torch.zeros(groups, count, dtype=torch.int64, device=x.device)
    ws = kernels.beam_select_workspace(x, beams, count)
    status = _native.lib().moe_beam_select(_native.BEAM_SELECT.pack(
        x.data_ptr(), x.shape[1], groups, beams, x.shape[1], 2, scores, count, out, parents.data_ptr(),
        tokens.data_ptr(), ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
    return status, parents, tokens


@gpu
def test_new_scores_may_take_the_old_ones_place():
    """Of the same shape; at another place over them they are refused."""
    from moeinfra_b200 import kernels

    x = _logits(40 * 4, 5000, torch.float32, 1)
    s = _scores(40, 4, 1)
    want = kernels.beam_select(x, s, 4)
    at = s.data_ptr()
    for out, count in ((at + 16, 4), (at - 16, 4), (at, 3), (at, 5)):
        assert _in_place(x, at, out, 4, count, 40)[0] == 1
    status, parents, tokens = _in_place(x, at, at, 4, 4, 40)
    kernels.check_device()
    assert status == 0
    assert torch.equal(s, want[0]) and torch.equal(parents, want[1]) and torch.equal(tokens, want[2])


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_as_many_tokens_as_are_served(dtype):
    from moeinfra_b200 import kernels

    x, s = _logits(4, 1 << 20, dtype, 11), _scores(2, 2, 11)
    x[1, -1] = x[3, 0] = 30.0
    got = kernels.beam_select(x, s, 64)
    kernels.check_device()
    _check(x, s, 64, got)
