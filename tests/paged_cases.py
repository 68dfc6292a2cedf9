"""Batches over a paged cache for the tests: tensors, and what 64 bits say."""
from __future__ import annotations

import torch

from oracle import paged as oracle

D = 128
SCALE = D ** -0.5


class Batch:
    """Sequences of lens[b] keys, the last new[b] of them new, in shuffled pages; nothing but NaN bits in unused slots."""

    def __init__(self, lens, new, heads, page_size, fp8=False, ragged=True, seed=0, device="cuda", extra_pages=2, spread=1.0):
        self.lens, self.new, self.page_size, self.fp8, self.ragged = list(lens), list(new), page_size, fp8, ragged
        self.hq, self.hkv = heads
        g = torch.Generator().manual_seed(seed)
        b = len(self.lens)
        needed = [-(-n // page_size) for n in self.lens]
        self.pages = sum(needed) + extra_pages
        order = torch.randperm(self.pages, generator=g).to(torch.int32)
        self.table = torch.full((b, max(needed + [1])), 2 ** 30, dtype=torch.int32)  # entries behind the end are never read
        at = 0
        for i, n in enumerate(needed):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.tokens = sum(self.new)
        self.cu = torch.tensor([sum(self.new[:i]) for i in range(b + 1)], dtype=torch.int32)

        def rows(*shape, by=0.5):
            return (torch.randn(*shape, generator=g) * by).to(torch.bfloat16)

        self.q = rows(self.tokens, self.hq, D, by=spread)
        self.kv = [rows(2, n, self.hkv, D, by=1.0) for n in self.lens]  # of every sequence, in order
        self.seq_lens = torch.tensor(self.lens, dtype=torch.int32)
        self.device = device

    def cache_tensors(self):
        """Cache tensors (k, v, k_scale, v_scale) on the CPU, every key of every sequence written by the oracle."""
        shape = (self.pages, self.page_size, self.hkv, D)
        out = []
        for c in range(2):
            if self.fp8:
                k = torch.full(shape, 0x7f, dtype=torch.uint8)
                s = torch.full((self.pages, self.hkv, self.page_size, D // 32), 255, dtype=torch.uint8)
            else:
                k = torch.full(shape, float("nan"), dtype=torch.bfloat16)
                s = None
            for i, n in enumerate(self.lens):
                j = torch.arange(n)
                page, slot = self.table[i].long()[j // self.page_size], j % self.page_size
                if self.fp8:
                    codes, e = oracle.quantise(self.kv[i][c])
                    k[page, slot] = codes
                    s[page, :, slot] = e
                else:
                    k[page, slot] = self.kv[i][c]
            out.append((k.view(torch.float8_e4m3fn) if self.fp8 else k, s))
        return out[0][0], out[1][0], out[0][1], out[1][1]

    def on(self, t):
        return None if t is None else t.to(self.device)

    def shaped(self, t):
        """[tokens, heads, D] as the call takes it."""
        return t if self.ragged else t.view(len(self.lens), self.new[0], *t.shape[1:])

    def expected(self, tensors, causal, scale=SCALE):
        """o [tokens, hq, D], lse [hq, tokens], mass of o, size of the scores."""
        k, v, ks, vs = tensors
        parts = []
        for i, n in enumerate(self.lens):
            kk = oracle.gather(k, ks, self.table[i], n, self.page_size)
            vv = oracle.gather(v, vs, self.table[i], n, self.page_size)
            parts.append(oracle.attend(self.q[self.cu[i]:self.cu[i + 1]], kk, vv, scale, causal))
        return (torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts], 1),
                torch.cat([p[2] for p in parts]), torch.cat([p[3] for p in parts], 1))


def bounds(o, mass, size):
    """How far o and lse may be off.

    o: probabilities are rounded to bf16 before a product summed in fp32, and the result is rounded: 2^-8 each, relative to
    sum p |v| and |o|, and 5 % for the exponentials and fp32 sums (tests/helpers.py: rounding_bound).
    lse: 8 sums of 16 products, each off by 2^-23 of the sum of magnitudes; the exponent's fma 2^-24 of its
    size, which that covers; ex2 and log 2^-21; adding n <= 2^13 terms in up to 2^8 fp32 steps per lane 2^-16."""
    from tests.helpers import rounding_bound

    return rounding_bound(mass, o), 2.0 ** -19 * size + 2.0 ** -16 + 2.0 ** -20


def check(batch, got_o, got_lse, want):
    o, lse, mass, size = want
    got_o, got_lse = got_o.double().cpu().reshape(o.shape), got_lse.double().cpu()
    if not batch.ragged:
        got_lse = got_lse.permute(1, 0, 2).reshape(lse.shape)
    tol_o, tol_lse = bounds(o, mass, size)
    assert not torch.isnan(got_o).any() and not torch.isnan(got_lse).any()
    none = torch.isinf(lse)
    assert torch.equal(torch.isinf(got_lse), none) and (got_lse[none] < 0).all()
    assert (got_o.permute(1, 0, 2)[none] == 0).all()
    off = (got_o - o).abs() - tol_o
    assert off.max().item() <= 0, f"o off by {(got_o - o).abs().max().item():.3g}, {off.max().item():.3g} over the bound"
    d = (got_lse - lse)[~none].abs() - tol_lse[~none]
    assert d.numel() == 0 or d.max().item() <= 0, f"lse {d.max().item():.3g} over the bound"
