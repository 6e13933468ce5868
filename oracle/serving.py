"""Paged serving in 64 bits on the CPU: the formulas of the kernels' rotation, cache and attention.

Each function also gives what a rounding bound needs (the sums of absolute values the rounded
quantities enter with), so a test's tolerance follows from the number formats.
"""
from __future__ import annotations

import torch

# Half a unit in the last place, relative: the largest rounding error of one value.
ROUNDING = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}


def rotary_table(positions: int, head_dim: int, theta: float = 1e6):
    """(cos, sin) fp32 [positions, head_dim / 2] of HF's default frequencies."""
    inv = theta ** (-torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim)
    angle = torch.outer(torch.arange(positions, dtype=torch.float64), inv)
    return angle.cos().float(), angle.sin().float()


def rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """x [tokens, heads, hd] by its tokens' rows of cos / sin [tokens, hd / 2]; float64."""
    a, b = x.double().chunk(2, dim=-1)
    c, s = cos.double()[:, None], sin.double()[:, None]
    return torch.cat((a * c - b * s, b * c + a * s), -1)


def gather_pages(pages: torch.Tensor, table_row: torch.Tensor, length: int) -> torch.Tensor:
    """The first ``length`` positions of a sequence: [kv_heads, length, hd]."""
    n, kv, size, hd = pages.shape
    at = table_row[:-(-length // size)].long()
    return pages[at].transpose(0, 1).reshape(kv, -1, hd)[:, :length]


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, causal: bool):
    """q [n, H, hd], k / v [m, KV, hd] of one sequence -> (out, bound part) float64 [n, H, hd].

    The last query sees all m keys when ``causal``; a query without keys gives zeros.  The second
    value is sum_j p_j |v_j|, and the third how far a score may be off when the products are summed
    in fp32: hd 2^-24 scale sum_i |q_i k_i|, its largest over the keys.
    """
    n, H, hd = q.shape
    m, KV = k.shape[:2]
    q, k, v = (t.double().transpose(0, 1) for t in (q, k, v))
    k, v = (t.repeat_interleave(H // KV, 0) for t in (k, v))
    if m == 0:
        z = torch.zeros(n, H, hd, dtype=torch.float64)
        return z, z, z[..., :1]
    s = q @ k.transpose(1, 2) * scale
    off = (q.abs() @ k.abs().transpose(1, 2) * scale).amax(-1, keepdim=True) * hd * 2.0 ** -24
    if causal:
        i = torch.arange(n)[:, None] + (m - n)
        s = s.masked_fill(torch.arange(m)[None] > i, float("-inf"))
    p = torch.softmax(s, -1)
    p = torch.where(torch.isneginf(s.amax(-1, keepdim=True)), 0.0, p)
    return tuple(t.transpose(0, 1) for t in (p @ v, p @ v.abs(), off))


def attention_bound(dtype: torch.dtype, out, weight, off):
    """Largest error of a kernel that rounds probabilities and outputs to ``dtype``.

    The output's rounding u |o|; a probability's own rounding u and twice the score's error (in
    the numerator and in the sum) on each p_j |v_j|; 2^-19 for the exponential (2 ulp), the fp32
    sums and the joins; the smallest steps of the formats.
    """
    u = ROUNDING[dtype]
    return u * out.abs() + (u + 2 * off + 2.0 ** -19) * weight + SMALLEST[dtype]


def sample(x, u: float, temperature: float, top_k: int, top_p: float, min_p: float):
    """One row of the sampler: (token, probability), in Python integers over float32 exponentials.

    The definition's exponential is fp32's, which libraries round differently in the last place;
    the third value says whether the token is sure all the same: every boundary it depends on is
    further off than all weights moved by one part in 2^21 could carry it.
    """
    import math

    import numpy as np

    x = np.asarray(x, np.float32) + np.float32(0)
    x = np.where(np.isnan(x), np.float32(-np.inf), x)
    m = x.max()
    order = sorted(range(len(x)), key=lambda i: (-x[i], i))
    if not temperature > 0 or top_k == 1:
        return order[0], 1.0, True
    with np.errstate(invalid="ignore", over="ignore"):
        d = np.where(x == m, np.float32(0), (x - m) / np.float32(temperature))
    e = np.exp(d.astype(np.float64)).astype(np.float32)
    w = [int(float(v) * 2.0 ** 40) for v in e]
    kept = order[:top_k] if 0 < top_k < len(x) else order
    sure = True
    if np.float32(top_p) < 1:
        total = sum(w[i] for i in kept)
        need = max(1, min(total, math.ceil(float(np.float32(top_p)) * total)))
        run, n = 0, 0
        while run < need:
            run += w[kept[n]]
            n += 1
        slack = total >> 21
        sure &= run - need > slack and need - (run - w[kept[n - 1]]) > slack
        kept = kept[:n]
    lim = min(np.float32(min_p), np.float32(1))
    sure &= all(abs(float(e[i]) - float(lim)) > 2e-6 * float(lim) for i in kept if e[i] != 1)
    kept = sorted(i for i in kept if e[i] >= lim)
    total = sum(w[i] for i in kept)
    r = max(0, min(total - 1, math.floor(float(np.float32(u)) * total)))
    run = 0
    for i in kept:
        if run + w[i] > r:
            sure &= run + w[i] - r > (total >> 21) and (r - run > (total >> 21) or run == 0)
            return i, w[i] / total, sure
        run += w[i]
    raise AssertionError("the sums cover every r")
