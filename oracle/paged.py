"""Keys and values in pages, in 64 bits on the CPU: what kv_cache_write, kv_cache_read and attn_fwd_paged compute.

Plain loops over sequences; values of e4m3 are found by comparing with the whole grid."""
from __future__ import annotations

import math

import torch

D = 128
BLOCK = 32

# The values of e4m3 from zero up: subnormals of step 2^-9, then three fraction bits, up to 448.
GRID = torch.tensor([i * 2.0 ** -9 for i in range(8)] +
                    [(1 + f / 8) * 2.0 ** e for e in range(-6, 9) for f in range(8) if (e, f) != (8, 7)], dtype=torch.float64)


def nearest_e4m3(x: torch.Tensor) -> torch.Tensor:
    """Codes (0..255) of the nearest e4m3 values; a tie goes to the even code, what is beyond 448 becomes that."""
    a = x.double().abs().clamp(max=448.0)
    hi = torch.searchsorted(GRID, a.contiguous()).clamp(max=len(GRID) - 1)
    lo = (hi - 1).clamp(min=0)
    up, down = GRID[hi] - a, a - GRID[lo]
    code = torch.where((up < down) | ((up == down) & (hi % 2 == 0)) | (a == GRID[hi]), hi, lo)
    return (code + torch.where(torch.signbit(x), 128, 0)).to(torch.uint8)


def code_values(codes: torch.Tensor) -> torch.Tensor:
    v = GRID[(codes & 127).long().clamp(max=len(GRID) - 1)]
    return torch.where(codes >= 128, -v, v)


def scale_exponents(x: torch.Tensor) -> torch.Tensor:
    """Per 32 values the least e in [-50, 64] with max|x| <= 448 * 2^e; 128 where a value is not finite."""
    most = x.double().unflatten(-1, (-1, BLOCK)).abs().amax(-1)
    e = torch.full(most.shape, 64.0, dtype=torch.float64)
    for k in range(63, -51, -1):
        e = torch.where(most <= 448.0 * 2.0 ** k, torch.full_like(e, k), e)
    return torch.where(torch.isfinite(most), e, torch.full_like(e, 128.0))


def quantise(x: torch.Tensor):
    """(codes, scale bytes) of rows [..., 128]."""
    e = scale_exponents(x)
    y = x.double().unflatten(-1, (-1, BLOCK)) * torch.exp2(-e).unsqueeze(-1)
    return nearest_e4m3(torch.nan_to_num(y)).flatten(-2), (e + 127).to(torch.uint8)


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    s = torch.exp2(scales.double() - 127)
    s = torch.where(scales >= 192, torch.full_like(s, math.nan), s)
    return (code_values(codes).unflatten(-1, (-1, BLOCK)) * s.unsqueeze(-1)).flatten(-2)


def gather(k, k_scale, table, length, page_size):
    """[length, heads, 128] in 64 bits: the first keys (or values) of one sequence.  k_scale: None for bf16."""
    j = torch.arange(length)
    page, slot = table.long()[j // page_size], j % page_size
    if k_scale is None:
        return k[page, slot].double()
    return values(k.view(torch.uint8)[page, slot], k_scale[page, :, slot])


def attend(q, k, v, scale, causal):
    """q [n, hq, D]; k, v [len, hkv, D] in 64 bits -> o, lse [hq, n], sum_j p_j |v_j|, max_j sum_d |q_d k_d|."""
    n, hq, _ = q.shape
    length, hkv, _ = k.shape
    q = q.double()
    group = hq // hkv
    kk, vv = (x.repeat_interleave(group, 1).permute(1, 0, 2) for x in (k, v))  # [hq, len, D]
    qq = q.permute(1, 0, 2)
    s = qq @ kk.transpose(1, 2) * scale
    if causal:
        hidden = torch.arange(length)[None] > torch.arange(n)[:, None] + length - n
        s = s.masked_fill(hidden, -math.inf)
    lse = torch.logsumexp(s, 2) if length else torch.full((hq, n), -math.inf, dtype=torch.float64)
    p = torch.where(torch.isfinite(lse)[..., None], torch.exp(s - lse[..., None]), torch.zeros_like(s))
    size = (qq.abs() @ kk.abs().transpose(1, 2)).amax(2) * scale if length else torch.zeros(hq, n, dtype=torch.float64)
    return (p @ vv).permute(1, 0, 2), lse, (p @ vv.abs()).permute(1, 0, 2), size
