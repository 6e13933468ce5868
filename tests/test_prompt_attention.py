"""Attention over packed prompts against its formula in 64 bits.

Tolerance: ``oracle.serving.attention_bound`` (derived from the formats' roundings).
"""
from __future__ import annotations

import pytest
import torch

from oracle import serving as ref

gpu = pytest.mark.gpu


def _offsets(lens):
    return torch.tensor([0] + lens).cumsum(0).int()


def _inputs(lens, lens_k, H, KV, hd, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(sum(lens), H, hd, generator=g).to(dtype)
    k, v = (torch.randn(sum(lens_k), KV, hd, generator=g).to(dtype) for _ in range(2))
    return q, k, v


def _run(q, k, v, lens, lens_k, causal=True, scale=None, **kw):
    from moeinfra_b200 import kernels

    same = lens is lens_k
    return kernels.prompt_attention(
        q.cuda(), k.cuda(), v.cuda(), _offsets(lens).cuda(), max(lens),
        cu_seqlens_k=None if same else _offsets(lens_k).cuda(),
        max_seqlen_k=None if same else max(lens_k), causal=causal, scale=scale, **kw)


def _check(q, k, v, lens, lens_k=None, causal=True, scale=None):
    from moeinfra_b200 import kernels

    lens_k = lens if lens_k is None else lens_k
    got = _run(q, k, v, lens, lens_k, causal, scale)
    kernels.check_device()
    a = c = 0
    for n, m in zip(lens, lens_k):
        want, weight, off = ref.attention(q[a:a + n], k[c:c + m], v[c:c + m],
                                          q.shape[2] ** -0.5 if scale is None else scale, causal)
        bound = ref.attention_bound(q.dtype, want, weight, off)
        err = (got[a:a + n].double().cpu() - want).abs()
        assert (err <= bound).all(), (n, m, float((err / bound).max()))
        a, c = a + n, c + m
    return got


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H,KV", [(4, 1), (2, 2), (6, 2), (7, 1), (8, 1), (32, 2), (32, 1)])
def test_heads_and_types(dtype, hd, H, KV):
    lens = [40, 1, 200, 129]
    _check(*_inputs(lens, lens, H, KV, hd, dtype, seed=H), lens)


@gpu
@pytest.mark.parametrize("lens", [[1], [2], [127], [128], [129], [255], [256], [257], [385],
                                  [1000], [0, 5, 0], [0], [300, 0, 0, 17, 256, 1, 128],
                                  list(range(1, 60)), [513] * 9, [1700, 3]])
@pytest.mark.parametrize("causal", [True, False])
def test_lengths(lens, causal):
    """Tiles of 128 rows and keys, blocks of 256 rows: their edges, one and zero tokens."""
    _check(*_inputs(lens, lens, 2, 1, 64, torch.float16, seed=len(lens)), lens, causal=causal)


@gpu
@pytest.mark.parametrize("lens,lens_k", [
    ([1, 1, 1], [300, 1, 128]), ([40, 7], [296, 7]), ([256, 130], [700, 131]),
    ([100, 20], [30, 0]), ([300], [1]), ([5, 400, 5], [0, 300, 260]), ([3], [0])])
@pytest.mark.parametrize("causal", [True, False])
def test_keys_of_other_lengths(lens, lens_k, causal):
    """Prompts that continue earlier keys, single tokens, and more queries than keys: rows that
    see nothing are zeros."""
    q, k, v = _inputs(lens, lens_k, 4, 2, 128, torch.bfloat16, seed=5)
    got = _check(q, k, v, lens, lens_k, causal)
    a = 0
    for n, m in zip(lens, lens_k):
        blind = n if m == 0 else max(0, n - m) if causal else 0
        assert not got[a:a + blind].any()
        a += n


@gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_other_sequences_have_no_effect(bad):
    """Infinities and NaN in the rows of the neighbours, which share tiles with a sequence's end."""
    lens = [100, 40, 200, 130]
    q, k, v = _inputs(lens, lens, 2, 1, 128, torch.float16, seed=1)
    clean = _run(q, k, v, lens, lens)
    for t in (q, k, v):
        t[100:140] = bad
    got = _run(q, k, v, lens, lens)
    for lo, hi in ((0, 100), (140, 470)):
        assert torch.equal(got[lo:hi], clean[lo:hi])


@gpu
def test_strides_and_streams():
    """q, k and v as views of one projection; a call on another stream."""
    from moeinfra_b200 import kernels

    lens, H, KV, hd = [150, 33], 4, 2, 64
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(sum(lens), H + 2 * KV, hd, generator=g).half()
    parts = [t.contiguous() for t in (qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:])]
    want = _check(*parts, lens)
    d, cu = qkv.cuda(), _offsets(lens).cuda()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = kernels.prompt_attention(d[:, :H], d[:, H:H + KV], d[:, H + KV:], cu, max(lens))
    s.synchronize()
    assert torch.equal(got, want)
    # Every second head of a wider tensor.
    wide = torch.randn(sum(lens), 2 * H, hd, generator=g).half()
    want = _check(wide[:, ::2].contiguous(), *parts[1:], lens)
    got = kernels.prompt_attention(wide.cuda()[:, ::2], d[:, H:H + KV], d[:, H + KV:], cu, max(lens))
    assert torch.equal(got, want)


@gpu
def test_growing_and_peaked_scores():
    """Scores that rise along the keys (each step raises the maximum, by less and by more than
    what is left standing), one key far above the rest, and all scores far below zero."""
    n, hd = 700, 64
    g = torch.Generator().manual_seed(0)
    v = torch.randn(n, 1, hd, generator=g).half()
    q = torch.zeros(n, 1, hd)
    q[..., 0] = 1.0
    ramps = [torch.linspace(0, 60, n), torch.linspace(0, 3, n), torch.linspace(60, 0, n),
             torch.full((n,), -500.0), torch.where(torch.arange(n) == 300, 12.0, 0.0),
             torch.where(torch.arange(n) % 128 == 0, 20.0, -3.0)]
    for ramp in ramps:
        k = torch.zeros(n, 1, hd)
        k[:, 0, 0] = ramp
        for causal in (True, False):
            _check(q.half(), k.half(), v, [n], causal=causal, scale=1.0)
            _check(q.bfloat16(), k.bfloat16(), v.bfloat16(), [n], causal=causal, scale=1.0)


@gpu
def test_a_captured_call_follows_its_offsets():
    from moeinfra_b200 import kernels

    q, k, v = (t.cuda() for t in _inputs([300], [300], 2, 1, 64, torch.float16))
    cu = _offsets([300, 0, 0]).cuda()
    kernels.prompt_attention(q, k, v, cu, 300)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kernels.prompt_attention(q, k, v, cu, 300)
    for lens in ([300, 0, 0], [1, 259, 40], [100, 100, 100]):
        cu.copy_(_offsets(lens))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, kernels.prompt_attention(q, k, v, cu, 300))


@gpu
def test_bad_offsets_are_reported():
    """Offsets that fall, leave the rows or exceed the stated length: that sequence's rows are not
    written, the others are right."""
    from moeinfra_b200 import kernels

    q, k, v = _inputs([200], [200], 2, 1, 64, torch.float16)
    want = _run(q[:60], k[:60], v[:60], [60], [60])
    for cu in ([0, 60, 20], [0, 60, 201], [0, 60, 1 << 30], [0, 60, 171], [0, 60, -4]):
        out = torch.full((200, 2, 64), 7.0, dtype=torch.float16, device="cuda")
        kernels.prompt_attention(q.cuda(), k.cuda(), v.cuda(), torch.tensor(cu).int().cuda(), 110,
                                 out=out)
        with pytest.raises(RuntimeError, match="out of range"):
            kernels.check_device()
        assert torch.equal(out[:60], want) and (out[60:] == 7).all()
    kernels.check_device()


def test_host_checks_precede_every_launch():
    from moeinfra_b200 import _native

    lib, f, odd = _native.lib(), 0x100000, 0x100008

    def attend(q=f, rows=10, seqs=2, H=4, KV=2, hd=128, dtype=0, scale=1.0, stride=None, out=f,
               max_q=8, k=f, head=None, ws=f, bytes_=16):
        return lib.moe_prompt_attention(_native.PROMPT_ATTENTION.pack(
            q, H * hd if stride is None else stride, hd if head is None else head, rows, k, KV * hd,
            hd, f, KV * hd, hd, rows, f, f, seqs, max_q, 8, H, KV, hd, 1, dtype, scale, out, ws,
            bytes_, 0))

    assert lib.moe_prompt_attention(None) == 1
    assert attend(rows=0) == 0 and attend(seqs=0) == 0 and attend(max_q=0) == 0
    assert attend(rows=-1) == 1 and attend(H=5) == 1 and attend(q=0) == 1 and attend(k=0) == 1
    assert attend(scale=0.0) == 1 and attend(scale=float("nan")) == 1 and attend(stride=8) == 1
    assert attend(head=64) == 1 and attend(seqs=-1) == 1
    assert attend(hd=96) == 2 and attend(dtype=2) == 2
    assert attend(ws=0) == 4 and attend(bytes_=15) == 4 and attend(ws=odd) == 5
    assert attend(q=odd) == 5 and attend(out=odd) == 5 and attend(stride=516) == 5


def test_wrapper_refuses_cpu_tensors():
    from moeinfra_b200 import kernels

    q = torch.zeros(4, 2, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        kernels.prompt_attention(q, q, q, torch.tensor([0, 4]).int(), 4)


@gpu
def test_wrapper_refuses_wrong_shapes_and_types():
    from moeinfra_b200 import kernels

    q = torch.zeros(4, 4, 64, dtype=torch.float16, device="cuda")
    kv = torch.zeros(4, 2, 64, dtype=torch.float16, device="cuda")
    cu = torch.tensor([0, 4]).int().cuda()

    def attend(q=q, k=kv, v=kv, cu=cu, **kw):
        return kernels.prompt_attention(q, k, v, cu, 4, **kw)

    attend()
    for bad in (dict(q=q.float()), dict(q=q[..., :48]), dict(k=kv.bfloat16()), dict(v=kv[:3]),
                dict(q=q[:, :3]), dict(cu=cu.long()), dict(cu=cu[:0]), dict(q=q[0]),
                dict(out=q.bfloat16()), dict(cu_seqlens_k=cu), dict(k=kv.transpose(1, 2)),
                dict(cu_seqlens_k=cu[:1], max_seqlen_k=4)):
        with pytest.raises(ValueError):
            attend(**bad)
    with pytest.raises(RuntimeError):
        attend(scale=0.0)
    with pytest.raises(ValueError, match="workspace"):
        attend(workspace=torch.zeros(8, dtype=torch.uint8, device="cuda"))


def _spoilt(q, k, v, lens, sure):
    """Runs the call; rows that ``sure`` marks must be NaN, the others within the usual bound of
    what the formula gives without the spoilt rows' keys having an effect."""
    from moeinfra_b200 import kernels

    got = _run(q, k, v, lens, lens).double().cpu()
    kernels.check_device()
    a = 0
    for n in lens:
        rows = slice(a, a + n)
        clean = [torch.nan_to_num(t[rows].double(), 0.0, 0.0, 0.0).to(t.dtype) for t in (q, k, v)]
        want, weight, off = ref.attention(*clean, q.shape[2] ** -0.5, True)
        bad = sure[rows]
        assert got[rows][bad].isnan().all()
        bound = ref.attention_bound(q.dtype, want, weight, off)
        assert ((got[rows] - want).abs() <= bound)[~bad].all()
        a += n


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_nan_of_a_key_or_query_reaches_the_rows_that_see_it(dtype, hd, bad):
    """At every place of a step's 80 or 96 keys; an infinite score has a NaN softmax too."""
    lens = [250, 40]
    for at in list(range(0, 100, 7)) + list(range(1, 97, 8)) + [95, 96, 97, 191, 249, 250, 289]:
        q, k, v = _inputs(lens, lens, 4, 2, hd, dtype, seed=at)
        q = q.abs() + 0.1  # inf: every score with the key is +inf
        k[at, 1] = bad
        n = torch.arange(290)
        sees = (n >= at) & ((n < 250) == (at < 250))
        sure = torch.zeros(290, 4, dtype=torch.bool)
        sure[sees, 2:] = True
        _spoilt(q, k, v, lens, sure)
    q, k, v = _inputs(lens, lens, 4, 2, hd, dtype, seed=1)
    sure = torch.zeros(290, 4, dtype=torch.bool)
    for at, h in ((0, 0), (17, 1), (100, 3), (249, 2), (251, 0)):
        q[at, h] = float("nan")
        sure[at, h] = True
    _spoilt(q, k, v, lens, sure)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128])
def test_scores_of_minus_infinity(dtype, hd):
    """One key of probability 0 leaves a row as if it were not there; with no other key it is 0 / 0."""
    inf, n = float("inf"), 200
    q, k, v = _inputs([n], [n], 2, 1, hd, dtype, seed=2)
    q[..., 0], k[..., 0] = 1.0, 0.0
    rest = torch.ones(n, dtype=torch.bool)
    for at in (0, 5, 8, 63, 130):
        kk = k.clone()
        kk[at, 0, 0] = -inf
        got = _run(q, kk, v, [n], [n]).double().cpu()
        assert got[:1].isnan().all() == (at == 0) and not got[1:].isnan().any()
        rest[:], rest[at] = True, False
        want, weight, off = ref.attention(q[-1:], k[rest], v[rest], hd ** -0.5, True)
        bound = ref.attention_bound(dtype, want, weight, off)
        assert ((got[-1:] - want).abs() <= bound).all()
    k[:, 0, 0] = -inf
    assert _run(q, k, v, [n], [n]).isnan().all()


@gpu
@pytest.mark.parametrize("hd", [64, 128])
def test_large_values_of_keys_not_seen_have_no_effect(hd):
    """bf16 values near the largest: a probability that is merely tiny would let them through."""
    n = 150
    q, k, v = _inputs([n], [n], 2, 1, hd, torch.bfloat16, seed=3)
    clean = _run(q, k, v, [n], [n])
    for at in (1, 8, 16, 79, 100):
        w = v.clone()
        w[at:] = 3e38
        got = _run(q, k, w, [n], [n])
        want, weight, off = ref.attention(q[:at], k[:at], v[:at], hd ** -0.5, True)
        bound = ref.attention_bound(torch.bfloat16, want, weight, off)
        assert ((got[:at].double().cpu() - want).abs() <= bound).all()
    assert torch.equal(clean, _run(q, k, v, [n], [n]))


def _value_spoilt(lens, lens_k, H, KV, hd, dtype, at, dims, bad):
    """Value row ``at`` of every KV head is ``bad`` in ``dims``: rows that see it are not finite there,
    all else is as the formula says."""
    from moeinfra_b200 import kernels

    q, k, v = _inputs(lens, lens_k, H, KV, hd, dtype, seed=at)
    spoilt = v.clone()
    spoilt[at, :, dims] = bad
    got = _run(q, k, spoilt, lens, lens_k).double().cpu()
    kernels.check_device()
    a = c = 0
    for n, m in zip(lens, lens_k):
        want, weight, off = ref.attention(q[a:a + n], k[c:c + m], v[c:c + m], hd ** -0.5, True)
        sees = (torch.arange(n) + m - n + c >= at) & (c <= at < c + m)
        odd = torch.zeros(n, H, hd, dtype=torch.bool)
        odd[sees, :, dims] = True
        mine = got[a:a + n]
        assert not mine[odd].isfinite().any()
        # The spoilt row counts in no other row, and in no other dim of the rows that see it.
        bound = ref.attention_bound(dtype, want, weight, off)
        assert ((mine - want).abs() <= bound)[~odd].all(), (at, n, m)
        a, c = a + n, c + m


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H,KV", [(8, 2), (1, 1), (16, 1), (3, 1)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_values_of_keys_not_seen_have_no_effect(dtype, hd, H, KV, bad):
    """Infinities and NaN among the values of later keys, which share tiles with the rows before."""
    for at in (0, 1, 40, 79, 80, 95, 96, 127, 128, 170, 255, 299, 300, 330):
        for dims in (slice(None), slice(3, 4)):
            _value_spoilt([300, 35], [300, 35], H, KV, hd, dtype, at, dims, bad)
    for at in (10, 333, 399, 400, 419):  # prompts that continue earlier keys; fewer keys than queries
        _value_spoilt([130, 40], [400, 20], H, KV, hd, dtype, at, slice(None), bad)


@gpu
def test_values_not_seen_in_strided_rows():
    from moeinfra_b200 import kernels

    lens, H, KV, hd = [150, 33], 4, 2, 64
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(sum(lens), H + 2 * KV, hd, generator=g).half().cuda()
    qkv[100, H + KV:] = float("inf")
    cu = _offsets(lens).cuda()
    q, k, v = qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:]
    got = kernels.prompt_attention(q, k, v, cu, max(lens))
    packed = kernels.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), cu, max(lens))
    assert torch.equal(got[:100], packed[:100]) and got[:100].isfinite().all()
    assert not got[100:150].isfinite().any() and torch.equal(got[150:], packed[150:])


@gpu
@pytest.mark.parametrize("H,KV", [(4, 1), (2, 2), (16, 1)])
@pytest.mark.parametrize("lens", [[5], [300, 1, 0, 64], [1 + i % 64 for i in range(1000)],
                                  [0] * 700 + [40] + [0] * 700, [9] * 500 + [3000] + [17] * 500,
                                  [0, 0, 0]])
def test_lengths_far_below_the_stated_maximum(H, KV, lens):
    from moeinfra_b200 import kernels

    q, k, v = (t.cuda() for t in _inputs(lens, lens, H, KV, 64, torch.float16, seed=len(lens)))
    cu = _offsets(lens).cuda()
    want = kernels.prompt_attention(q, k, v, cu, max(max(lens), 1))
    most = 131072 if len(lens) * H < 4000 else 32768
    for stated in (max(lens) + 1, 4096, most):
        assert torch.equal(kernels.prompt_attention(q, k, v, cu, stated), want)
    kernels.check_device()
    # Offsets that are wrong anywhere are still reported, those of empty sequences too.
    bad_k = cu.clone()
    bad_k[-1] = q.shape[0] + 1
    kernels.prompt_attention(q, k, v, cu, most, cu_seqlens_k=bad_k, max_seqlen_k=most)
    if q.shape[0]:
        with pytest.raises(RuntimeError, match="out of range"):
            kernels.check_device()
    kernels.check_device()


@gpu
def test_a_stated_maximum_that_takes_long_to_walk():
    """2 million blocks of which the last 2000 or so have rows (walking them took 15 ms): no wait runs
    out."""
    from moeinfra_b200 import _native, kernels

    lens, H = [1 + i % 30 for i in range(1000)], 16
    q, k, v = (t.cuda() for t in _inputs(lens, lens, H, 1, 64, torch.float16))
    cu = _offsets(lens).cuda()
    want = kernels.prompt_attention(q, k, v, cu, 30)
    old = _native.wait_limit_ns()
    _native.set_wait_limit_ns(5_000_000)
    try:
        got = kernels.prompt_attention(q, k, v, cu, 32768)
        kernels.check_device()
    finally:
        _native.set_wait_limit_ns(old)
    assert torch.equal(got, want)


@gpu
def test_values_not_seen_of_a_long_prompt():
    """Rows that are computed again over 20000 keys keep no wait of the other warps too long."""
    from moeinfra_b200 import kernels

    n, H, KV, hd = 20000, 16, 1, 128
    g = torch.Generator(device="cuda").manual_seed(8)
    q = torch.randn(n, H, hd, device="cuda", generator=g).bfloat16()
    kv = torch.randn(n, 2 * KV, hd, device="cuda", generator=g).bfloat16()
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    clean = kernels.prompt_attention(q, kv[:, :KV], kv[:, KV:], cu, n)
    kv[n - 3, KV:, 7] = float("inf")
    got = kernels.prompt_attention(q, kv[:, :KV], kv[:, KV:], cu, n)
    kernels.check_device()
    assert not got[n - 3:, :, 7].isfinite().any()
    # The same row twice, its probabilities rounded to 16 bits or not: two roundings and theirs.
    # sum_j p_j |v_j| <= max |v| < 6, a probability's rounding is 2^-8 of it at most.
    got[n - 3:, :, 7] = clean[n - 3:, :, 7]
    assert got.isfinite().all()
    assert float((got.float() - clean.float()).abs().max()) <= 6 * 2 ** -8
