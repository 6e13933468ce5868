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
