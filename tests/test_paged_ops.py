"""Rotation + paged append and paged attention against their formulas in 64 bits.

Tolerances: a rotated value is one rounding of an fp32 expression of two products (three fp32
roundings of terms at most |x| + |y|); attention's bound is ``oracle.serving.attention_bound``.
"""
from __future__ import annotations

import inspect
import random

import pytest
import torch

from oracle import serving as ref

gpu = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def _cache(pages, kv, page, hd, dtype, seed, fill=None, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    if fill is None:
        return torch.randn(pages, kv, page, hd, generator=g).to(dtype).to(device)
    return torch.full((pages, kv, page, hd), fill, dtype=dtype, device=device)


def _table(lens, page, seed, width=None):
    """A block table over shuffled pages; entries past a sequence's last page are -1."""
    need = [-(-n // page) for n in lens]
    order = list(range(sum(need) + 2))
    random.Random(seed).shuffle(order)
    table = torch.full((len(lens), max(max(need), 1) if width is None else width), -1,
                       dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    return table, sum(need) + 2


# -- rope_append --------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KV,hd,page", [(4, 2, 64, 16), (32, 8, 128, 16), (7, 7, 128, 48),
                                          (28, 4, 64, 32), (1, 1, 128, 1)])
@pytest.mark.parametrize("prompt", [False, True])
def test_rope_append(dtype, H, KV, hd, page, prompt):
    from moeinfra_b200 import kernels

    lens = [1, 2 * page + 1, page, 37, 3]
    table, n_pages = _table(lens, page, 1)
    kp, vp = (_cache(n_pages, KV, page, hd, dtype, 0, fill=7.0) for _ in range(2))
    want_k, want_v = kp.double().cpu(), vp.double().cpu()
    cos, sin = ref.rotary_table(max(lens), hd)
    if prompt:
        seq = torch.cat([torch.full((n,), b) for b, n in enumerate(lens)])
        pos = torch.cat([torch.arange(n) for n in lens])
        order = torch.randperm(len(pos), generator=torch.Generator().manual_seed(3))
        seq, pos = seq[order], pos[order]  # any order of tokens
    else:
        seq, pos = torch.arange(len(lens)), torch.tensor(lens) - 1
    T = len(pos)
    g = torch.Generator().manual_seed(2)
    # Rows of a wider buffer: the projection's rows may be strided.
    wide = torch.randn(T, (H + 2 * KV) * hd + 64, generator=g).to(dtype)
    qkv = wide.cuda()[:, :(H + 2 * KV) * hd]
    packed = torch.empty(T, KV, hd, dtype=dtype, device="cuda")
    q = kernels.rope_append(qkv, cos.cuda(), sin.cuda(), pos.int().cuda(), table.cuda(), kp, vp, H,
                            seq_ids=seq.int().cuda() if prompt else None,
                            k_out=packed if prompt else None)
    kernels.check_device()
    if prompt:
        at = table[seq, pos // page].long().cuda()
        assert torch.equal(packed, kp[at, :, (pos % page).cuda()])
    x = wide[:, :(H + 2 * KV) * hd].view(T, H + 2 * KV, hd)
    rot = ref.rotate(x[:, :H + KV], cos[pos], sin[pos])
    size = x[:, :H + KV].double().abs()
    size = (size[..., :hd // 2] + size[..., hd // 2:]).repeat(1, 1, 2)
    bound = ref.ROUNDING[dtype] * rot.abs() + 2.0 ** -22 * size + ref.SMALLEST[dtype]
    assert ((q.double().cpu() - rot[:, :H]).abs() <= bound[:, :H]).all()
    tol = torch.zeros_like(want_k)
    for t in range(T):
        p, r = int(table[seq[t], pos[t] // page]), int(pos[t]) % page
        want_k[p, :, r], want_v[p, :, r] = rot[t, H:], x[t, H + KV:].double()
        tol[p, :, r] = bound[t, H:]
    assert ((kp.double().cpu() - want_k).abs() <= tol).all()  # other slots keep their 7.0
    assert torch.equal(vp.double().cpu(), want_v)


@gpu
def test_rope_append_leaves_padding_and_refuses_bad_places():
    """A negative position is padding; a position, sequence or page out of range touches nothing
    and is reported."""
    from moeinfra_b200 import kernels

    H, KV, hd, page = 4, 2, 64, 16
    cos, sin = (t.cuda() for t in ref.rotary_table(40, hd))
    table = torch.tensor([[0, 1], [2, 99], [-5, 1]], dtype=torch.int32, device="cuda")
    kp, vp = (_cache(3, KV, page, hd, torch.float16, 0, fill=7.0) for _ in range(2))
    qkv = torch.randn(1, (H + 2 * KV) * hd, device="cuda").half()

    def run(pos, seq):
        one = [torch.tensor([v], dtype=torch.int32, device="cuda") for v in (pos, seq)]
        return kernels.rope_append(qkv, cos, sin, one[0], table, kp, vp, H, seq_ids=one[1])

    packed = torch.full((1, KV, hd), 7.0, dtype=torch.float16, device="cuda")
    none = torch.tensor([-1], dtype=torch.int32, device="cuda")
    kernels.rope_append(qkv, cos, sin, none, table, kp, vp, H, k_out=packed)
    assert not run(-1, 0).any() and not packed.any()
    kernels.check_device()
    for pos, seq in [(40, 0), (33, 0), (0, 3), (0, -1), (20, 1), (0, 2)]:
        assert not run(pos, seq).any()
        with pytest.raises(RuntimeError, match="out of range"):
            kernels.check_device()
    assert (kp == 7).all() and (vp == 7).all()
    kernels.check_device()


@gpu
def test_rope_append_takes_no_tokens_and_other_streams():
    from moeinfra_b200 import kernels

    H, KV, hd, page = 4, 2, 64, 16
    cos, sin = (t.cuda() for t in ref.rotary_table(8, hd))
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    kp, vp = (_cache(1, KV, page, hd, torch.float16, 0, fill=0.0) for _ in range(2))
    none = torch.empty(0, (H + 2 * KV) * hd, device="cuda", dtype=torch.float16)
    pos = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert kernels.rope_append(none, cos, sin, pos, table, kp, vp, H).shape == (0, H, hd)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        qkv = torch.ones(1, (H + 2 * KV) * hd, device="cuda", dtype=torch.float16)
        q = kernels.rope_append(qkv, cos, sin, torch.zeros(1, dtype=torch.int32, device="cuda"),
                                table, kp, vp, H)
    s.synchronize()
    assert (q == 1).all() and (kp[0, :, 0] == 1).all() and (vp[0, :, 0] == 1).all()
    assert not kp[0, :, 1:].any()


# -- paged_attention ----------------------------------------------------------------------------

def _check_paged(q, kp, vp, table, lens, scale=None):
    from moeinfra_b200 import kernels

    got = kernels.paged_attention(q.cuda(), kp.cuda(), vp.cuda(), table.cuda(),
                                  torch.tensor(lens, dtype=torch.int32, device="cuda"), scale)
    kernels.check_device()
    sc = q.shape[2] ** -0.5 if scale is None else scale
    for b, n in enumerate(lens):
        k, v = (ref.gather_pages(p.cpu(), table[b], n).transpose(0, 1) for p in (kp, vp))
        want, weight, off = ref.attention(q[b:b + 1].cpu(), k, v, sc, causal=False)
        bound = ref.attention_bound(q.dtype, want, weight, off)
        err = (got[b:b + 1].double().cpu() - want).abs()
        assert (err <= bound).all(), (b, n, float((err / bound).max()))
    return got


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H,KV", [(32, 8), (4, 4), (7, 1), (28, 4), (16, 1), (40, 2), (24, 1)])
def test_paged_attention_heads(dtype, hd, H, KV):
    """Groups of 1 to 24 heads; lengths at the edges of chunks and pages."""
    lens = [1, 15, 16, 17, 0, 33, 64, 65, 100]
    table, n = _table(lens, 16, 5)
    g = torch.Generator().manual_seed(H + hd)
    q = torch.randn(len(lens), H, hd, generator=g).to(dtype)
    kp, vp = (_cache(n, KV, 16, hd, dtype, s) for s in (1, 2))
    _check_paged(q, kp, vp, table, lens)


@gpu
@pytest.mark.parametrize("lens,page,width", [
    ([1], 16, 64), ([1024], 16, None), ([1025], 16, None), ([3000], 16, None),
    ([5000, 1, 0, 700], 64, None), ([0, 0, 0], 16, 70), ([2047, 2048, 2049], 48, None),
    ([257] * 40, 32, None), ([31, 4000] * 20, 128, None), ([1] * 300, 16, None),
    ([0] * 200 + [1500] + [0] * 90, 16, None)])
def test_paged_attention_lengths(lens, page, width):
    """One CTA per unit and cut lines, units over many CTAs, whole units inside a warp's share,
    empty sequences before, between and after."""
    H, KV, hd = 8, 2, 64
    table, n = _table(lens, page, 6, width)
    g = torch.Generator().manual_seed(len(lens))
    q = torch.randn(len(lens), H, hd, generator=g).half()
    kp, vp = (_cache(n, KV, page, hd, torch.float16, s) for s in (3, 4))
    got = _check_paged(q, kp, vp, table, lens)
    for b, m in enumerate(lens):
        assert m or not got[b].any()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KV,hd", [(8, 4, 64), (24, 4, 128), (48, 4, 128)])
@pytest.mark.parametrize("width", [80, 128, 140])
def test_paged_attention_many_sequences(dtype, H, KV, hd, width):
    """More sequences than processors, in tables of every split's width; the lengths decide
    nothing about the split, so they range from none to all of a table."""
    page, lens = 16, [0, 1, 15, 16, 17, 1025, 1280, 79, 0] + [3 + 7 * i for i in range(40)]
    table, n = _table(lens, page, 12, width)
    kp, vp = (_cache(n, KV, page, hd, dtype, s) for s in (13, 14))
    q = torch.randn(len(lens), H, hd, generator=torch.Generator().manual_seed(15)).to(dtype)
    _check_paged(q, kp, vp, table, lens)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H,KV", [(16, 1), (12, 1), (24, 1), (32, 2), (8, 1)])
def test_paged_attention_wide_groups_over_a_cut_line(dtype, hd, H, KV):
    """Groups of 8 to 24 heads over tables too long for a CTA per unit."""
    page, lens = 16, [3000, 17, 0, 1025, 16]
    table, n = _table(lens, page, 21)
    g = torch.Generator().manual_seed(H + hd)
    q = torch.randn(len(lens), H, hd, generator=g).to(dtype)
    kp, vp = (_cache(n, KV, page, hd, dtype, s) for s in (22, 23))
    _check_paged(q, kp, vp, table, lens)


@gpu
@pytest.mark.parametrize("hd,H", [(64, 16), (128, 16), (64, 4)])
def test_paged_attention_of_as_many_sequences_as_fit(hd, H):
    page, lens = 16, [(37 * i) % 49 for i in range(4095)]
    table, n = _table(lens, page, 24)
    g = torch.Generator().manual_seed(25)
    q = torch.randn(len(lens), H, hd, generator=g).half()
    kp, vp = (_cache(n, 1, page, hd, torch.float16, s) for s in (26, 27))
    got = _check_paged(q, kp, vp, table, lens)
    assert not got[::49].any()  # those of no length


@gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("lens", [[5, 20], [1500, 16]])
def test_paged_attention_ignores_what_lies_past_the_end(bad, lens):
    from moeinfra_b200 import kernels

    H, KV, hd, page = 8, 2, 128, 32
    table, n = _table(lens, page, 8)
    g = torch.Generator().manual_seed(1)
    q = torch.randn(len(lens), H, hd, generator=g).half().cuda()
    kp, vp = (_cache(n, KV, page, hd, torch.float16, s) for s in (5, 6))
    at = torch.tensor(lens, dtype=torch.int32, device="cuda")
    clean = kernels.paged_attention(q, kp, vp, table.cuda(), at)
    used = {int(p) for row in table for p in row if p >= 0}
    for p in range(n):
        if p not in used:
            kp[p], vp[p] = bad, bad
    for b, m in enumerate(lens):
        if m % page:
            last = int(table[b, m // page])
            kp[last, :, m % page:], vp[last, :, m % page:] = bad, bad
    assert torch.equal(kernels.paged_attention(q, kp, vp, table.cuda(), at), clean)


@gpu
def test_paged_attention_of_a_peaked_and_a_faint_softmax():
    """One key far above the others (their probabilities near fp16's smallest), and scores far
    below zero: nothing underflows to a wrong sum."""
    H, KV, hd, page, m = 4, 1, 64, 16, 600
    table, n = _table([m, m], page, 2)
    kp = torch.zeros(n, KV, page, hd)
    vp = torch.randn(n, KV, page, hd, generator=torch.Generator().manual_seed(0))
    q = torch.zeros(2, H, hd)
    q[:, :, 0] = 1.0
    for b, base in ((0, 0.0), (1, -300.0)):
        kp[table[b, :-(-m // page)].long(), 0, :, 0] = base
        kp[int(table[b, 3]), 0, 5, 0] = base + 11.0
    _check_paged(q.half(), kp.half(), vp.half(), table, [m, m], scale=1.0)


@gpu
def test_paged_attention_strided_inputs_shared_pages_and_repeats():
    """Pages with the keys and values side by side, rows of q from a wider buffer, one page in
    two sequences; the same call twice gives the same bits."""
    from moeinfra_b200 import kernels

    H, KV, hd, page, lens = 8, 2, 128, 16, [40, 2000, 33]
    table, n = _table(lens, page, 9)
    table[2, 0] = table[0, 0]
    both = _cache(2 * n, KV, page, hd, torch.bfloat16, 7).view(n, 2, KV, page, hd)
    kp, vp = both[:, 0], both[:, 1]
    wide = torch.randn(3, 2 * H, hd, generator=torch.Generator().manual_seed(4)).bfloat16()
    q = wide.cuda()[:, H:]
    got = kernels.paged_attention(q, kp, vp, table.cuda(), torch.tensor(lens).int().cuda())
    packed = _check_paged(wide[:, H:].contiguous(), kp.contiguous(), vp.contiguous(), table, lens)
    assert torch.equal(got, packed)
    again = kernels.paged_attention(q, kp, vp, table.cuda(), torch.tensor(lens).int().cuda())
    assert torch.equal(got, again)


@gpu
def test_paged_attention_follows_lengths_in_a_graph():
    """A captured call reads lengths and pages when it is replayed."""
    from moeinfra_b200 import kernels

    H, KV, hd, page = 8, 2, 64, 16
    lens = [300, 2100]
    table, n = _table([2400, 2400], page, 3)
    kp, vp = (_cache(n, KV, page, hd, torch.float16, s) for s in (8, 9))
    q = torch.randn(2, H, hd, generator=torch.Generator().manual_seed(5)).half().cuda()
    tab, at = table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")
    kernels.paged_attention(q, kp, vp, tab, at)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kernels.paged_attention(q, kp, vp, tab, at)
    for lens in ([300, 2100], [0, 17], [2400, 1]):
        at.copy_(torch.tensor(lens))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, kernels.paged_attention(q, kp, vp, tab, at))


@gpu
def test_paged_attention_reports_bad_lengths_and_pages():
    from moeinfra_b200 import kernels

    H, KV, hd, page = 4, 2, 64, 16
    kp, vp = (_cache(2, KV, page, hd, torch.float16, s) for s in (8, 9))
    q = torch.ones(1, H, hd, dtype=torch.float16, device="cuda")
    for table, n in (([0, 1], 33), ([0, 1], -1), ([0, 7], 32), ([-1, 0], 3)):
        kernels.paged_attention(q, kp, vp, torch.tensor([table], dtype=torch.int32, device="cuda"),
                                torch.tensor([n], dtype=torch.int32, device="cuda"))
        with pytest.raises(RuntimeError, match="out of range"):
            kernels.check_device()
    kernels.check_device()


@gpu
def test_paged_attention_past_two_to_the_31_elements():
    """Pages whose elements lie past 2^31 (and bytes past 2^32) of the cache."""
    from moeinfra_b200 import kernels

    H, KV, hd, page = 2, 1, 128, 64
    n = (1 << 31) // (KV * page * hd) + 40
    kp = torch.empty(n, KV, page, hd, dtype=torch.float16, device="cuda")
    vp = torch.empty_like(kp)
    far, near = list(range(n - 20, n)), list(range(20))
    g = torch.Generator(device="cuda").manual_seed(0)
    for p in (kp, vp):
        p[n - 20:] = torch.randn(20, KV, page, hd, device="cuda", generator=g).half()
        p[:20] = torch.randn(20, KV, page, hd, device="cuda", generator=g).half()
    table = torch.tensor([far, near], dtype=torch.int32)
    lens = [20 * page - 3, 20 * page]
    q = torch.randn(2, H, hd, generator=torch.Generator().manual_seed(1)).half()
    got = kernels.paged_attention(q.cuda(), kp, vp, table.cuda(), torch.tensor(lens).int().cuda())
    kernels.check_device()
    for b in range(2):
        at = table[b].long().cuda()
        small = torch.arange(20, dtype=torch.int32)
        k, v = (ref.gather_pages(p[at].cpu(), small, lens[b]).transpose(0, 1) for p in (kp, vp))
        want, weight, off = ref.attention(q[b:b + 1], k, v, hd ** -0.5, causal=False)
        bound = ref.attention_bound(torch.float16, want, weight, off)
        assert ((got[b:b + 1].double().cpu() - want).abs() <= bound).all()


# -- refusals -----------------------------------------------------------------------------------

def test_host_checks_precede_every_launch():
    """No pointer below is dereferenced: every refusal comes before the launch."""
    from moeinfra_b200 import _native

    lib, f, odd = _native.lib(), 0x100000, 0x100008

    def append(T=4, hd=128, page=16, dtype=0, stride=None, H=4, KV=2, p=f, pages=f, kstride=None,
               k_out=0):
        elems = KV * page * hd
        return lib.moe_rope_append(_native.ROPE_APPEND.pack(
            pages, f, elems if kstride is None else kstride, elems, 4, KV, page, hd, dtype, f, 4, 4, 4,
            p, (H + 2 * KV) * hd if stride is None else stride, f, f, 8, f, 0, T, H, f, k_out, 0))

    assert append(T=0) == 0 and lib.moe_rope_append(None) == 1
    assert append(T=-1) == 1 and append(p=0) == 1 and append(H=0) == 1
    assert append(stride=100) == 1 and append(kstride=64) == 1
    assert append(hd=96) == 2 and append(dtype=2) == 2
    assert append(k_out=odd) == 5 and append(p=odd) == 5 and append(pages=odd) == 5 and append(stride=1028) == 5

    need = lib.moe_paged_attention_workspace_size(4, 8, 16, 8, 2, 128)
    assert need > 0 and lib.moe_paged_attention_workspace_size(4, 8, 16, 8, 2, 96) == 0

    def attend(seqs=4, hd=128, page=16, H=8, KV=2, dtype=0, scale=1.0, q=f, ws=f, bytes_=need,
               qs=None):
        elems = KV * page * hd
        return lib.moe_paged_attention(_native.PAGED_ATTENTION.pack(
            f, f, elems, elems, 9, KV, page, hd, dtype, f, 8, seqs, 8, q,
            H * hd if qs is None else qs, H, f, scale, f, ws, bytes_, 0))

    assert attend(seqs=0) == 0 and lib.moe_paged_attention(None) == 1
    assert attend(H=7) == 1 and attend(scale=0.0) == 1 and attend(scale=float("nan")) == 1
    assert attend(scale=float("inf")) == 1 and attend(q=0) == 1 and attend(qs=64) == 1
    assert attend(hd=256) == 2 and attend(page=24) == 2 and attend(dtype=2) == 2
    assert attend(seqs=4096) == 2
    assert attend(bytes_=need - 1) == 4 and attend(ws=0) == 4
    assert attend(q=odd) == 5 and attend(ws=odd) == 5
    assert _native.status_string(8) != "unknown status"


@pytest.mark.parametrize("heads,kv,hd", [(32, 8, 128), (16, 1, 64), (17, 1, 128), (4, 4, 64)])
def test_a_workspace_serves_smaller_tables_too(heads, kv, hd):
    """Around 64 and 128 chunks of 16 positions, and the number of processors, the split changes."""
    from moeinfra_b200 import _native

    size = _native.lib().moe_paged_attention_workspace_size
    most = size(64, 400, 16, heads, kv, hd)
    assert most > 4096
    for seqs in [1, 2, 4, 9, 18, 19, 20, 37, 38, 63, 64]:
        for pages in [0, 1, 11, 12, 63, 64, 65, 127, 128, 129, 400]:
            assert 0 < size(seqs, pages, 16, heads, kv, hd) <= most


def test_lines_too_long_for_32_bits_are_refused():
    """16 sequences in tables of 134217727 pages of 16: 2^31 - 16 chunks.  Fewer sequences get as
    far as the check of the workspace."""
    from moeinfra_b200 import _native

    lib, f = _native.lib(), 0x100000

    def attend(seqs, pages, hd=128):
        return lib.moe_paged_attention(_native.PAGED_ATTENTION.pack(
            f, f, 16 * hd, 16 * hd, 9, 1, 16, hd, 0, f, pages, seqs, pages, f, hd, 1, f, 1.0, f, f, 0,
            0))

    assert attend(16, 134217727) == 2
    assert attend(8, 134217727) == 4 and attend(15, 134217727) == 4


def test_wrappers_refuse_cpu_tensors():
    from moeinfra_b200 import kernels

    kp = torch.zeros(2, 2, 16, 64, dtype=torch.float16)
    table = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        kernels.paged_attention(torch.zeros(1, 4, 64, dtype=torch.float16), kp, kp, table,
                                torch.ones(1, dtype=torch.int32))
    with pytest.raises(ValueError):
        kernels.paged_attention(torch.zeros(1, 4, 64), kp.float(), kp.float(), table,
                                torch.ones(1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="no CPU path"):
        kernels.rope_append(torch.zeros(1, 512, dtype=torch.float16), torch.zeros(4, 32),
                            torch.zeros(4, 32), torch.zeros(1, dtype=torch.int32), table, kp, kp, 4)


@gpu
def test_wrappers_refuse_wrong_shapes_and_types():
    from moeinfra_b200 import kernels

    kp = torch.zeros(2, 2, 16, 64, dtype=torch.float16, device="cuda")
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    at = torch.ones(1, dtype=torch.int32, device="cuda")
    q = torch.zeros(1, 4, 64, dtype=torch.float16, device="cuda")

    def attend(q=q, k=kp, v=kp, table=table, at=at, **kw):
        return kernels.paged_attention(q, k, v, table, at, **kw)

    attend()
    for bad in (dict(q=q.bfloat16()), dict(q=q[..., :32]), dict(q=q[:, :3]), dict(at=at.long()),
                dict(table=table.long()), dict(v=kp[:1]), dict(k=kp.float(), v=kp.float()),
                dict(q=q.expand(2, 4, 64)), dict(k=kp.transpose(0, 2), v=kp.transpose(0, 2)),
                dict(out=q.float())):
        with pytest.raises(ValueError):
            attend(**bad)
    with pytest.raises(RuntimeError):
        attend(scale=-1.0)
    odd = torch.zeros(2, 2, 24, 64, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError, match="multiple of 16"):
        attend(k=odd, v=odd)
    cos = torch.ones(4, 32, device="cuda")
    qkv = torch.zeros(2, 512, dtype=torch.float16, device="cuda")
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="sequences"):  # two tokens, one sequence, no seq_ids
        kernels.rope_append(qkv, cos, cos, pos, table, kp, kp, 4)
    for bad in (dict(qkv=qkv[:, :448]), dict(pos=pos.long()), dict(cos=cos[:, :16]),
                dict(pos=pos[:1])):
        args = dict(qkv=qkv, cos=cos, pos=pos) | bad
        with pytest.raises(ValueError):
            kernels.rope_append(args["qkv"], args["cos"], cos, args["pos"], table, kp, kp, 4,
                                seq_ids=pos)


@gpu
def test_a_callers_workspace_is_checked():
    """One in host memory, on another device, too small or with gaps is refused before the launch."""
    from moeinfra_b200 import kernels

    kp = torch.randn(2, 2, 16, 64, device="cuda").half()
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    at = torch.full((1,), 9, dtype=torch.int32, device="cuda")
    q = torch.randn(1, 4, 64, device="cuda").half()
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")

    def paged(ws):
        return kernels.paged_attention(q, kp, kp, table, at, workspace=ws)

    def prompt(ws):
        return kernels.prompt_attention(q, q[:, :2], q[:, 2:], cu, 1, workspace=ws)

    own = kernels.paged_attention_workspace(table, 16, 4, 2, 64)
    for call in (paged, prompt):
        assert torch.equal(call(own), call(None))
        for bad in (own.cpu(), own[:8], torch.zeros(2, own.numel(), device="cuda").t()):
            with pytest.raises(ValueError, match="workspace"):
                call(bad)
        with pytest.raises(TypeError, match="workspace"):
            call(own.data_ptr())


def _one_step(device):
    """Arguments of each serving operator by name, for one sequence."""
    def at(t, dtype=torch.float16):
        return t.to(dtype).to(device)

    g = torch.Generator().manual_seed(1)
    one, i32, f32 = torch.ones(1), torch.int32, torch.float32
    pages = at(torch.randn(2, 2, 16, 64, generator=g))
    cache = dict(k_pages=pages, v_pages=pages.clone(), block_table=at(0 * one[None], i32))
    q = torch.randn(1, 4, 64, generator=g)
    return {
        "rope_append": cache | dict(
            qkv=at(torch.randn(1, 512, generator=g)), cos=at(torch.rand(4, 32), f32),
            sin=at(torch.rand(4, 32), f32), positions=at(2 * one, i32), num_heads=4),
        "paged_attention": cache | dict(q=at(q), lengths=at(9 * one, i32)),
        "prompt_attention": dict(q=at(q), k=at(q[:, :2]), v=at(q[:, 2:]), max_seqlen=1,
                                 cu_seqlens=at(torch.arange(2), i32)),
        "sample_tokens": dict(logits=at(q[0]), uniforms=at(torch.rand(4), f32),
                              temperature=at(torch.ones(4), f32), top_k=at(torch.zeros(4), i32),
                              top_p=at(torch.ones(4), f32), min_p=at(torch.zeros(4), f32)),
        "paged_attention_workspace": dict(block_table=cache["block_table"], page_size=16,
                                          num_heads=4, kv_heads=2, head_dim=64),
    }


@pytest.mark.parametrize("name", ["rope_append", "paged_attention", "prompt_attention",
                                  "sample_tokens"])
def test_arguments_by_name_reach_the_checks(name):
    from moeinfra_b200 import kernels

    args = _one_step("cpu")[name]
    with pytest.raises(RuntimeError, match="no CPU path"):
        getattr(kernels, name)(**args)
    missing = next(iter(inspect.signature(getattr(kernels, name)).parameters))
    del args[missing]
    with pytest.raises(TypeError, match=missing):
        getattr(kernels, name)(**args)


@gpu
@pytest.mark.parametrize("name", ["rope_append", "paged_attention", "prompt_attention",
                                  "sample_tokens", "paged_attention_workspace"])
def test_arguments_by_name_and_by_place(name):
    from moeinfra_b200 import kernels

    fn, args = getattr(kernels, name), _one_step("cuda")[name]
    names = [n for n in inspect.signature(fn).parameters if n in args]
    by_place = [args[n] for n in names]
    got, want = fn(**args), fn(*by_place)
    half = fn(by_place[0], **{n: args[n] for n in names[1:]})
    for out in (got, half):
        pairs = zip(out, want) if isinstance(want, tuple) else [(out, want)]
        assert all(torch.equal(a, b) for a, b in pairs)


@gpu
def test_a_cache_without_heads_is_refused():
    from moeinfra_b200 import kernels

    none = torch.zeros(2, 0, 16, 64, dtype=torch.float16, device="cuda")
    at = torch.ones(1, dtype=torch.int32, device="cuda")
    q = torch.zeros(1, 4, 64, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError, match="KV heads"):
        kernels.paged_attention(q, none, none, at[None], at)
    with pytest.raises(ValueError, match="KV heads"):
        kernels.prompt_attention(q, q[:, :0], q[:, :0], torch.arange(2).int().cuda(), 1)
