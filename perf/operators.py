"""Cases of the paged-serving operators: their inputs, plain forms, exact values and work.

The operators are one decode engine's chain: ``rope_append`` (rotate q and k, write k and v into
the paged cache), ``prompt_attention`` (packed prompts), ``paged_attention`` (one new token per
sequence over the pages) and ``sample_tokens``.  With ``own`` false, :func:`run` computes a case in
elementary torch operations in 32 bits, rounded once; with ``own`` true it calls the framework.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
WEIGHT_SCALE = float(1 << 40)  # fixed point of the sampler's weights


def listed():
    return [
        # One sequence decoding, 32 query / 8 KV heads of 128: a step's rotation and cache write.
        {"name": "append one token", "op": "rope_append", "dtype": "fp16", "seqs": 1, "lo": 72,
         "hi": 72, "prompt": False, "heads": 32, "kv": 8, "hd": 128, "page": 16, "lens_seed": 1},
        # A decode batch of 64 sequences between 512 and 640 tokens.
        {"name": "append a batch", "op": "rope_append", "dtype": "bf16", "seqs": 64, "lo": 512,
         "hi": 640, "prompt": False, "heads": 32, "kv": 8, "hd": 128, "page": 64, "lens_seed": 2},
        # Prefill of 64 prompts of up to 512 tokens, packed.
        {"name": "append prompts", "op": "rope_append", "dtype": "fp16", "seqs": 64, "lo": 129,
         "hi": 512, "prompt": True, "heads": 32, "kv": 8, "hd": 128, "page": 16, "lens_seed": 3},
        # One chat in decode after a 40-token prompt: latency counts.
        {"name": "decode one short", "op": "paged_attention", "dtype": "fp16", "seqs": 1, "lo": 72,
         "hi": 72, "heads": 32, "kv": 8, "hd": 128, "page": 16, "lens_seed": 4},
        # A serving batch: 64 sequences, 512 prompt tokens and up to 128 decoded ones.
        {"name": "decode a batch", "op": "paged_attention", "dtype": "fp16", "seqs": 64, "lo": 512,
         "hi": 640, "heads": 32, "kv": 8, "hd": 128, "page": 16, "lens_seed": 5},
        # Long documents: few sequences, the cache's length is the work; odd lengths.
        {"name": "decode long", "op": "paged_attention", "dtype": "bf16", "seqs": 4, "lo": 65537,
         "hi": 131071, "heads": 32, "kv": 8, "hd": 128, "page": 64, "lens_seed": 6},
        # One 40-token prompt: time to first token.
        {"name": "prompt short", "op": "prompt_attention", "dtype": "fp16", "seqs": 1, "lo": 40,
         "hi": 40, "extra": 0, "heads": 32, "kv": 8, "hd": 128, "lens_seed": 7},
        # Prefill of 64 ragged prompts of up to 512 tokens.
        {"name": "prompts ragged", "op": "prompt_attention", "dtype": "fp16", "seqs": 64, "lo": 129,
         "hi": 512, "extra": 0, "heads": 32, "kv": 8, "hd": 128, "lens_seed": 8},
        # One long document.
        {"name": "prompt long", "op": "prompt_attention", "dtype": "bf16", "seqs": 1, "lo": 8192,
         "hi": 8192, "extra": 0, "heads": 32, "kv": 8, "hd": 128, "lens_seed": 9},
        # One chat, nucleus sampling over a vocabulary of 32000.
        {"name": "sample one", "op": "sample_tokens", "dtype": "fp16", "rows": 1, "vocab": 32000,
         "mix": False},
        # A batch whose requests carry different parameters (greedy ones among them).
        {"name": "sample a batch", "op": "sample_tokens", "dtype": "fp16", "rows": 64,
         "vocab": 32000, "mix": True},
        # A large batch over a wide vocabulary, fp32 logits.
        {"name": "sample wide", "op": "sample_tokens", "dtype": "fp32", "rows": 256,
         "vocab": 131072, "mix": True},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["rope_append", "paged_attention", "prompt_attention", "sample_tokens"])
    if op == "sample_tokens":
        vocab = _spread(rng, 4000, 131072)
        return {"op": op, "dtype": rng.choice(["fp16", "bf16", "fp32"]),
                "rows": _spread(rng, 1, 256), "vocab": vocab, "mix": rng.random() < 0.7}
    heads, kv = rng.choice([(32, 8), (32, 8), (32, 32), (16, 2), (28, 4), (8, 1), (4, 2)])
    case = {"op": op, "dtype": rng.choice(["fp16", "bf16"]), "heads": heads, "kv": kv,
            "hd": rng.choice([64, 128]), "lens_seed": rng.randrange(1 << 20)}
    if op == "rope_append":
        prompt = rng.random() < 0.5
        seqs = _spread(rng, 1, 64 if prompt else 256)
        hi = _spread(rng, 1, 512 if prompt else 2048)
        case.update(seqs=seqs, lo=max(1, hi // 4), hi=hi, prompt=prompt,
                    page=rng.choice([16, 32, 64, 128]))
    elif op == "paged_attention":
        seqs = _spread(rng, 1, 256)
        hi = _spread(rng, 1, min(131071, 4 * 98304 * 8 // (seqs * kv)))
        case.update(seqs=seqs, lo=max(1, hi // 4), hi=hi, page=rng.choice([16, 32, 64, 128]))
    else:
        seqs = _spread(rng, 1, 64)
        most = int(math.sqrt(8192 * 8192 * 32 / (seqs * heads)) / 1.25)
        hi = _spread(rng, 1, min(8192, most))
        # Sometimes the prompt continues keys that an earlier chunk left (extra of them a sequence).
        extra = rng.choice([0, 0, hi // 4])
        case.update(seqs=seqs, lo=max(1, hi // 4), hi=hi, extra=extra)
    return case


def _lengths(case):
    """The sequences' lengths: a property of the case, not of the seed."""
    rng = random.Random(case["lens_seed"])
    n = [rng.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]
    n[0] = case["hi"]
    return n


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, dtype, g):
    return torch.randn(shape, dtype=dtype, device="cuda", generator=g)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return _int32(cu)


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


def prepare(case, seed):
    g = _gen(seed)
    op, dt = case["op"], DTYPES[case["dtype"]]
    if op == "sample_tokens":
        return _prepare_sampling(case, dt, g)
    lens = _lengths(case)
    H, KV, hd = case["heads"], case["kv"], case["hd"]
    st = {"op": op, "H": H, "KV": KV, "hd": hd, "dtype": dt}
    if op == "prompt_attention":
        nk = [n + case["extra"] for n in lens]
        st["lens"], st["lens_k"] = lens, nk
        st["max"], st["max_k"] = max(lens), max(nk)
        st["cu"] = _offsets(lens)
        st["cu_k"] = _offsets(nk) if case["extra"] else None
        st["q"] = _randn((sum(lens), H, hd), dt, g)
        # k and v come as views of one projection's output, as the fused q/k/v product leaves them.
        kv = _randn((sum(nk), 2 * KV, hd), dt, g)
        st["k"], st["v"] = kv[:, :KV], kv[:, KV:]
        return st
    table, total = _pages(lens, case["page"], g)
    st["table"], st["page"] = table, case["page"]
    if op == "paged_attention":
        st["k_pages"] = _randn((total, KV, case["page"], hd), dt, g)
        st["v_pages"] = _randn((total, KV, case["page"], hd), dt, g)
        st["q"] = _randn((case["seqs"], H, hd), dt, g)
        st["lengths"] = _int32(lens)
        return st
    st["k_pages"] = torch.zeros((total, KV, case["page"], hd), dtype=dt, device="cuda")
    st["v_pages"] = torch.zeros_like(st["k_pages"])
    if case["prompt"]:
        cu = _offsets(lens)
        seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"),
                                      torch.tensor(lens, device="cuda")).to(torch.int32)
        st["seq_ids"] = seq
        st["positions"] = torch.arange(sum(lens), device="cuda", dtype=torch.int32) - cu[seq.long()]
    else:
        st["seq_ids"] = None
        st["positions"] = _int32([n - 1 for n in lens])
    st["qkv"] = _randn((st["positions"].numel(), (H + 2 * KV) * hd), dt, g)
    inv = 1e6 ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
    angle = torch.arange(max(lens), device="cuda", dtype=torch.float64)[:, None] * inv[None, :]
    st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
    return st


def _prepare_sampling(case, dt, g):
    B, V = case["rows"], case["vocab"]
    # A language model's logits: a broad bulk and a few hundred candidates that stand out.
    x = 2.0 * torch.randn((B, V), device="cuda", generator=g)
    stand_out = torch.rand((B, V), device="cuda", generator=g) < 200 / V
    boost = 3.0 + 2.5 * torch.randn((B, V), device="cuda", generator=g).abs()
    x += stand_out * boost
    st = {"op": "sample_tokens", "logits": x.to(dt),
          "uniforms": torch.rand(B, device="cuda", generator=g)}
    if case["mix"]:
        r = torch.arange(B, device="cuda") % 8
        st["temperature"] = torch.tensor([0.8, 1.0, 0.0, 0.7, 1.3, 1.0, 0.6, 1.0],
                                         device="cuda")[r].contiguous()
        st["top_k"] = torch.tensor([0, 50, 0, 40, 0, 0, 1000, 0], device="cuda",
                                   dtype=torch.int32)[r].contiguous()
        st["top_p"] = torch.tensor([0.95, 1.0, 1.0, 0.9, 1.0, 0.99, 0.8, 1.0],
                                   device="cuda")[r].contiguous()
        st["min_p"] = torch.tensor([0.0, 0.0, 0.0, 0.0, 0.05, 0.0, 0.01, 0.0],
                                   device="cuda")[r].contiguous()
    else:
        st["temperature"] = torch.full((B,), 0.8, device="cuda")
        st["top_k"] = torch.zeros(B, dtype=torch.int32, device="cuda")
        st["top_p"] = torch.full((B,), 0.95, device="cuda")
        st["min_p"] = torch.zeros(B, device="cuda")
    return st


def run(state):
    return (_run_own if own else _PLAIN[state["op"]])(state)


def _run_own(st):
    from moeinfra_b200 import kernels

    op = st["op"]
    if op == "rope_append":
        q = kernels.rope_append(st["qkv"], st["cos"], st["sin"], st["positions"], st["table"],
                                st["k_pages"], st["v_pages"], st["H"], seq_ids=st["seq_ids"])
        return {"q": q, "k_pages": st["k_pages"], "v_pages": st["v_pages"]}
    if op == "paged_attention":
        return {"o": kernels.paged_attention(st["q"], st["k_pages"], st["v_pages"], st["table"],
                                             st["lengths"])}
    if op == "prompt_attention":
        return {"o": kernels.prompt_attention(st["q"], st["k"], st["v"], st["cu"], st["max"],
                                              cu_seqlens_k=st["cu_k"], max_seqlen_k=st["max_k"])}
    tokens, probs = kernels.sample_tokens(st["logits"], st["uniforms"], st["temperature"],
                                          st["top_k"], st["top_p"], st["min_p"])
    return {"tokens": tokens, "probs": probs}


# -- plain forms ------------------------------------------------------------------------------

def _rotate(x, cos, sin):
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)


def _plain_rope_append(st):
    H, KV, hd, page = st["H"], st["KV"], st["hd"], st["page"]
    T = st["positions"].numel()
    pos = st["positions"].long()
    seq = torch.arange(T, device="cuda") if st["seq_ids"] is None else st["seq_ids"].long()
    x = st["qkv"].view(T, H + 2 * KV, hd)
    rot = _rotate(x[:, :H + KV].float(), st["cos"][pos][:, None], st["sin"][pos][:, None])
    rot = rot.to(st["dtype"])
    at = st["table"][seq, pos // page].long()
    st["k_pages"][at, :, pos % page] = rot[:, H:]
    st["v_pages"][at, :, pos % page] = x[:, H + KV:]
    return {"q": rot[:, :H].contiguous(), "k_pages": st["k_pages"], "v_pages": st["v_pages"]}


def _plain_paged_attention(st):
    H, KV, hd, page = st["H"], st["KV"], st["hd"], st["page"]
    B, P = st["table"].shape
    at = st["table"].clamp(min=0).long()
    keys = st["k_pages"][at].transpose(1, 2).reshape(B, KV, P * page, hd).float()
    vals = st["v_pages"][at].transpose(1, 2).reshape(B, KV, P * page, hd).float()
    q = st["q"].float().view(B, KV, H // KV, hd)
    s = (q @ keys.transpose(2, 3)) / math.sqrt(hd)
    seen = torch.arange(P * page, device="cuda")[None, :] < st["lengths"][:, None]
    s = s.masked_fill(~seen[:, None, None], float("-inf"))
    e = torch.exp(s - s.amax(-1, keepdim=True))
    o = (e @ vals) / e.sum(-1, keepdim=True)
    return {"o": o.reshape(B, H, hd).to(st["dtype"])}


def _padded(x, cu, longest):
    """Packed rows as [sequence, position, ...] (rows past a sequence's end repeat others)."""
    at = cu[:-1, None].long() + torch.arange(longest, device="cuda")[None, :]
    return x[at.clamp(max=x.shape[0] - 1)]


def _plain_prompt_attention(st):
    H, KV, hd, L, M = st["H"], st["KV"], st["hd"], st["max"], st["max_k"]
    cu = st["cu"]
    cu_k = cu if st["cu_k"] is None else st["cu_k"]
    n, nk = (cu[1:] - cu[:-1])[:, None, None], (cu_k[1:] - cu_k[:-1])[:, None, None]
    B = n.shape[0]
    q = _padded(st["q"], cu, L).float().transpose(1, 2).reshape(B, KV, H // KV * L, hd)
    keys = _padded(st["k"], cu_k, M).float().transpose(1, 2)
    vals = _padded(st["v"], cu_k, M).float().transpose(1, 2)
    s = (q @ keys.transpose(2, 3)).view(B, KV, H // KV, L, M)
    i = torch.arange(L, device="cuda")[None, :, None]
    j = torch.arange(M, device="cuda")[None, None, :]
    hidden = (j > i + (nk - n)) | (j >= nk)
    s = s.mul_(1.0 / math.sqrt(hd)).masked_fill_(hidden[:, None, None], float("-inf"))
    e = torch.exp_(s.sub_(s.amax(-1, keepdim=True)))
    o = (e.view(B, KV, H // KV * L, M) @ vals).view(B, KV, H // KV, L, hd)
    o = (o / e.sum(-1, keepdim=True)).reshape(B, H, L, hd).transpose(1, 2)
    real = torch.arange(L, device="cuda")[None, :] < n[:, 0]
    return {"o": o[real].to(st["dtype"])}


def _plain_sample_tokens(st):
    x = st["logits"].float() + 0.0
    B, V = x.shape
    x = x.masked_fill(x.isnan(), float("-inf"))
    greedy = (st["temperature"] == 0)[:, None]
    T = st["temperature"][:, None].masked_fill(greedy, 1.0)
    k = st["top_k"][:, None].long()
    k = torch.where(greedy, 1, torch.where(k > 0, k, V))
    top = x.amax(-1, keepdim=True)
    e = torch.exp(torch.where(x == top, 0.0, (x - top) / T))
    w = (e * WEIGHT_SCALE).long()
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    w_sorted, e_sorted = w.gather(1, order), e.gather(1, order)
    keep = torch.arange(V, device="cuda")[None, :] < k
    cum = (w_sorted * keep).cumsum(-1)
    total = cum[:, -1:]
    p = st["top_p"][:, None]
    need = torch.where(p < 1.0, torch.ceil(p.double() * total.double()).long(), total)
    keep &= cum - w_sorted < need.clamp(min=1)
    keep &= e_sorted >= st["min_p"][:, None]
    kept = torch.zeros_like(w).scatter_(1, order, w_sorted * keep)
    cum = kept.cumsum(-1)
    total = cum[:, -1:]
    r = torch.floor(st["uniforms"][:, None].double() * total.double()).long()
    r = torch.minimum(r, total - 1)
    tokens = (cum > r).long().argmax(-1)
    probs = kept.gather(1, tokens[:, None]).double() / total.double()
    return {"tokens": tokens, "probs": probs[:, 0].float()}


_PLAIN = {"rope_append": _plain_rope_append, "paged_attention": _plain_paged_attention,
          "prompt_attention": _plain_prompt_attention, "sample_tokens": _plain_sample_tokens}


# -- the definition in 64 bits -----------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    return {"rope_append": _exact_rope_append, "paged_attention": _exact_paged_attention,
            "prompt_attention": _exact_prompt_attention,
            "sample_tokens": _exact_sample_tokens}[case["op"]](case, st)


def _exact_rope_append(case, st):
    """Each pair (i, i + hd/2) as a complex number times exp(i position inv_freq)."""
    H, KV, hd, page = st["H"], st["KV"], st["hd"], st["page"]
    T = st["positions"].numel()
    x = st["qkv"].double().view(T, H + 2 * KV, 2, hd // 2)
    pos = st["positions"].long()
    turn = torch.complex(st["cos"].double(), st["sin"].double())[pos][:, None]
    y = torch.complex(x[:, :H + KV, 0], x[:, :H + KV, 1]) * turn
    y = torch.cat((y.real, y.imag), -1)
    seq = range(T) if st["seq_ids"] is None else st["seq_ids"].tolist()
    seq = torch.tensor(list(seq), device="cuda")
    slot = st["table"].long()[seq, torch.div(pos, page, rounding_mode="floor")] * page + pos % page
    out = {"q": y[:, :H].contiguous()}
    for name, rows in (("k_pages", y[:, H:]), ("v_pages", x[:, H + KV:].flatten(2))):
        flat = torch.zeros((st["k_pages"].shape[0] * page, KV, hd), dtype=torch.float64, device="cuda")
        flat.index_copy_(0, slot, rows.contiguous())
        out[name] = flat.view(-1, page, KV, hd).transpose(1, 2).contiguous()
    return out


def _softmax_rows(s, v):
    return torch.softmax(s, dim=-1) @ v


def _exact_paged_attention(case, st):
    H, KV, hd, page = st["H"], st["KV"], st["hd"], st["page"]
    out = torch.empty((case["seqs"], H, hd), dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(case)):
        at = st["table"][b, :-(-n // page)].long()
        k, v = (st[name][at].double().transpose(0, 1).flatten(1, 2)[:, :n]
                for name in ("k_pages", "v_pages"))
        q = st["q"][b].double().view(KV, H // KV, hd)
        out[b] = _softmax_rows(torch.einsum("kgd,knd->kgn", q, k) * hd ** -0.5, v).view(H, hd)
    return {"o": out}


def _exact_prompt_attention(case, st):
    H, KV, hd = st["H"], st["KV"], st["hd"]
    out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    a = c = 0
    for n, nk in zip(st["lens"], st["lens_k"]):
        hidden = torch.ones((n, nk), dtype=torch.bool, device="cuda").triu(nk - n + 1)
        for j in range(KV):
            q = st["q"][a:a + n, j * (H // KV):(j + 1) * (H // KV)].double().transpose(0, 1)
            k, v = st["k"][c:c + nk, j].double(), st["v"][c:c + nk, j].double()
            s = (q @ k.T * hd ** -0.5).masked_fill_(hidden, float("-inf"))
            out[a:a + n, j * (H // KV):(j + 1) * (H // KV)] = _softmax_rows(s, v).transpose(0, 1)
        a, c = a + n, c + nk
    return {"o": out}


def _exact_sample_tokens(case, st):
    """Row by row in 64-bit floats; the token has no computed value, its probability has."""
    probs = []
    for b in range(case["rows"]):
        x = st["logits"][b].double()
        T, k = float(st["temperature"][b]), int(st["top_k"][b])
        if T == 0:
            probs.append(torch.ones((), dtype=torch.float64, device="cuda"))
            continue
        p, order = torch.softmax(x / T, 0).sort(descending=True, stable=True)
        n = min(k, p.numel()) if k > 0 else p.numel()
        p = p[:n] / p[:n].sum()
        before = p.cumsum(0) - p
        kept = (before < float(st["top_p"][b])) & (p >= float(st["min_p"][b]) * p[0])
        index, at = order[:n][kept].sort()
        q = p[kept][at] / p[kept].sum()
        i = (q.cumsum(0) > float(st["uniforms"][b])).long().argmax()
        probs.append(q[i])
    return {"tokens": None, "probs": torch.stack(probs)}


def work(case):
    """Each input read once and each output written once; multiply-adds as two."""
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "sample_tokens":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * e + case["rows"] * (5 * 4 + 12), "flops": 4 * n}
    lens = _lengths(case)
    H, KV, hd = case["heads"], case["kv"], case["hd"]
    if case["op"] == "rope_append":
        T = sum(lens) if case["prompt"] else case["seqs"]
        rows = max(lens) if case["prompt"] else len(set(lens))
        return {"bytes": 2 * T * (H + 2 * KV) * hd * e + rows * hd * 4 + T * 12,
                "flops": 3 * T * (H + KV) * hd}
    if case["op"] == "paged_attention":
        pages = sum(-(-n // case["page"]) for n in lens)
        return {"bytes": sum(lens) * 2 * KV * hd * e + 2 * case["seqs"] * H * hd * e + 4 * pages
                + 4 * case["seqs"], "flops": 4 * sum(lens) * H * hd}
    x = case["extra"]
    pairs = sum(n * x + n * (n + 1) // 2 for n in lens)
    return {"bytes": (2 * sum(lens) * H + 2 * (sum(lens) + x * len(lens)) * KV) * hd * e,
            "flops": 4 * pairs * H * hd}
