"""What is timed of the paged K/V cache: writing it (bf16 or e4m3 with shared power-of-two scales), reading it back, and
attention of new tokens over it.

A case is a batch of sequences whose keys and values lie in pages.  `batch` sequences hold between `shortest` and
`longest` keys each, the new ones included; each has between `fewest` and `most` new tokens.  The lengths follow from the
case alone, the values, the order of the pages and the queries from the seed.  Head dimension 128 is what the library
takes.
"""
from __future__ import annotations

import math
import random

import torch

own = False

D = 128
BLOCK = 32  # values that share a scale
SCALE = D ** -0.5

# (query heads, K/V heads): the layouts of the benchmark and of the tests, and a group that is no power of two
HEADS = ((32, 32), (16, 16), (8, 8), (32, 8), (16, 4), (8, 2), (4, 2), (16, 1), (14, 2))


def listed():
    return [
        # one new token for each of 32 sequences goes into the cache: a serving step, launches and latency
        dict(name="write_step", kind="write", fp8=True, batch=32, shortest=1, longest=2000, fewest=1, most=1, hkv=8, page=16),
        # three prompts of odd lengths go into the cache in bf16
        dict(name="write_prompts_bf16", kind="write", fp8=False, batch=3, shortest=1500, longest=9001, fewest=1500, most=9001, hkv=8, page=64),
        # a long prompt is quantised as it is written
        dict(name="write_prompt_fp8", kind="write", fp8=True, batch=2, shortest=32768, longest=32768, fewest=32768, most=32768, hkv=8, page=64),
        # cached prefixes of odd lengths back into one packed buffer
        dict(name="read_ragged_bf16", kind="read", fp8=False, batch=5, shortest=1, longest=1025, fewest=1, most=1, hkv=4, page=16),
        # a long cached prefix back in bf16, for the ring schedules, which take packed keys and values
        dict(name="read_fp8", kind="read", fp8=True, batch=2, shortest=30001, longest=32768, fewest=1, most=1, hkv=8, page=32),
        # one token of one short conversation: the smallest call
        dict(name="token_short", kind="attend", fp8=False, batch=1, shortest=777, longest=777, fewest=1, most=1, hq=8, hkv=2, page=16, causal=True, ragged=False),
        # a serving step: one token for each of 64 sequences of many lengths
        dict(name="tokens_bf16", kind="attend", fp8=False, batch=64, shortest=50, longest=8192, fewest=1, most=1, hq=32, hkv=8, page=16, causal=True, ragged=False),
        # the same with the quantised cache, which holds twice the keys
        dict(name="tokens_fp8", kind="attend", fp8=True, batch=64, shortest=100, longest=16384, fewest=1, most=1, hq=32, hkv=8, page=16, causal=True, ragged=False),
        # five drafted tokens at once for few sequences, no grouped heads
        dict(name="drafts", kind="attend", fp8=False, batch=4, shortest=3000, longest=6001, fewest=5, most=5, hq=16, hkv=16, page=32, causal=True, ragged=False),
        # a chunk of a long prompt against what is cached of it
        dict(name="chunk_bf16", kind="attend", fp8=False, batch=1, shortest=32768, longest=32768, fewest=2048, most=2048, hq=32, hkv=8, page=64, causal=True, ragged=False),
        # prompts in chunks and single tokens in one batch, quantised cache
        dict(name="mixed_fp8", kind="attend", fp8=True, batch=16, shortest=700, longest=8192, fewest=1, most=512, hq=32, hkv=8, page=16, causal=True, ragged=True),
        # decoder tokens over an encoder's states of another length (not causal)
        dict(name="cross", kind="attend", fp8=False, batch=8, shortest=200, longest=1500, fewest=100, most=448, hq=16, hkv=16, page=128, causal=False, ragged=True),
    ]


def _log_size(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    # half as they come (odd ones among them), the others in the multiples that programs use
    step = rng.choice((1, 1, 16, 64)) if n >= 64 else 1
    return max(lo, n // step * step)


def draw(rng):
    limit = {"bytes": max(work(c)["bytes"] for c in listed()), "flops": max(work(c)["flops"] for c in listed())}
    while True:
        kind = rng.choice(("write", "read", "attend", "attend", "attend"))
        hq, hkv = rng.choice(HEADS)
        c = dict(kind=kind, fp8=rng.random() < 0.5, batch=_log_size(rng, 1, 64), hkv=hkv, page=rng.choice((16, 16, 32, 64, 128, 24)))
        c["longest"] = _log_size(rng, 1, 32768)
        c["shortest"] = rng.choice((c["longest"], max(1, c["longest"] // 2), 1))
        if kind == "attend":
            c.update(hq=hq, causal=rng.random() < 0.8, ragged=rng.random() < 0.5)
            c["most"] = rng.choice((1, 1, rng.randint(2, 8), _log_size(rng, 9, 2048)))
            if c["causal"] and c["most"] > c["longest"]:
                continue
        else:
            c["most"] = 1 if kind == "read" or rng.random() < 0.4 else c["longest"]
        c["fewest"] = c["most"] if not c.get("ragged", True) else rng.choice((1, c["most"]))
        w = work(c)
        # what the plain form holds at one time: scores in 32 bits, or the cache
        held = c["batch"] * c["longest"] * (c["most"] * hq if kind == "attend" else 1) * 4
        if w["bytes"] <= limit["bytes"] and w["flops"] <= limit["flops"] and held <= 9 << 30 and c["batch"] * c["longest"] * hkv <= 8 << 20:
            return c


def _lengths(c):
    """(keys, new tokens) of every sequence: the longest and the shortest first, the others in between."""
    rng = random.Random(c["batch"] * 1000003 + c["longest"])
    keys = [c["longest"], c["shortest"]] + [rng.randint(c["shortest"], c["longest"]) for _ in range(c["batch"])]
    keys = keys[:c["batch"]]
    new = [c["most"], c["fewest"]] + [rng.randint(c["fewest"], c["most"]) if rng.random() < 0.5 else c["fewest"] for _ in range(c["batch"])]
    new = new[:c["batch"]]
    if c["kind"] == "write":  # new tokens are among the keys
        new = [min(n, k) for n, k in zip(new, keys)]
    return keys, new


def work(c):
    keys, new = _lengths(c)
    row = D + D // BLOCK if c["fp8"] else 2 * D  # bytes of a cached head of one token
    if c["kind"] == "write":
        t = sum(new) * c["hkv"] * 2
        return {"bytes": t * (2 * D + row), "flops": t * D * (3 if c["fp8"] else 0)}
    if c["kind"] == "read":
        t = sum(keys) * c["hkv"] * 2
        return {"bytes": t * (2 * D + row), "flops": t * D * (1 if c["fp8"] else 0)}
    pairs, seen = 0, 0
    for k, n in zip(keys, new):
        if c["causal"]:
            first = max(0, n - k)  # rows before it see nothing
            pairs += sum(k - n + 1 + i for i in range(first, n))
        else:
            pairs += k * n
        seen += k
    return {"bytes": seen * c["hkv"] * 2 * row + sum(new) * c["hq"] * (4 * D + 4), "flops": 4 * D * c["hq"] * pairs}


# -- the plain forms -----------------------------------------------------------------------------------------------------
def _quantise(x):
    """Codes (e4m3) and scale bytes of rows [..., D]: the least power of two 2^e, -50 <= e <= 64, with max|x| <= 448 * 2^e per 32 values."""
    b = x.float().unflatten(-1, (D // BLOCK, BLOCK))
    m, e = torch.frexp(b.abs().amax(-1, keepdim=True))
    e = torch.where(m > 0, e - 9 + (m > 0.875), torch.full_like(e, -50)).clamp(-50, 64)
    codes = torch.ldexp(b, -e).clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes.flatten(-2), (e + 127).to(torch.uint8).squeeze(-1)


def _values(codes, scales):
    """The values that codes and scale bytes stand for."""
    return torch.ldexp(codes.float().unflatten(-1, (D // BLOCK, BLOCK)), scales.int().unsqueeze(-1) - 127).flatten(-2)


def _slots(s, positions, sequence):
    """Page and slot of keys at `positions` of `sequence` (tensors of one shape)."""
    return s["page_table"][sequence, positions // s["page"]].long(), positions % s["page"]


def _cached(s, which):
    """[batch, longest, hkv, D] in 32 bits: every sequence's cached keys or values (behind a sequence's end: page 0's)."""
    j = torch.arange(s["longest"], device="cuda").expand(s["batch"], -1)
    j = torch.where(j < s["seq_lens"][:, None], j, 0)
    page, slot = _slots(s, j, torch.arange(s["batch"], device="cuda")[:, None])
    rows = s[which].view(torch.uint8)[page, slot].view(s[which].dtype)
    if not s["fp8"]:
        return rows.float()
    return _values(rows, s[which + "_scale"][page, :, slot])


def _token_places(s):
    """Sequence and position of every new token [T]."""
    token = torch.arange(s["tokens"], dtype=torch.int32, device="cuda")
    sequence = torch.searchsorted(s["cu_seqlens"][1:], token, right=True)
    return sequence, token - s["cu_seqlens"][sequence + 1] + s["seq_lens"][sequence]


def _write_plain(s):
    sequence, position = _token_places(s)
    page, slot = _slots(s, position, sequence)
    for which, x in (("k", s["new_k"]), ("v", s["new_v"])):
        if s["fp8"]:
            codes, scales = _quantise(x)
            s[which].view(torch.uint8)[page, slot] = codes.view(torch.uint8)
            s[which + "_scale"][page, :, slot] = scales
        else:
            s[which][page, slot] = x
    return _cache_of(s)


def _cache_of(s):
    return [s["k"], s["v"]] + ([s["k_scale"], s["v_scale"]] if s["fp8"] else [])


def _read_plain(s):
    there = (torch.arange(s["longest"], device="cuda") < s["seq_lens"][:, None])[None, :, :, None, None]
    kv = torch.stack([_cached(s, "k"), _cached(s, "v")]).to(torch.bfloat16)
    torch.where(there, kv, s["out"], out=s["out"])
    return s["out"]


def _attend_plain(s):
    b, n, hq, hkv = s["batch"], s["most"], s["hq"], s["hkv"]
    group = hq // hkv
    if s["ragged"]:  # to [batch, most, heads, D]
        i = torch.arange(n, device="cuda")[None]
        new = (s["cu_seqlens"][1:] - s["cu_seqlens"][:-1])[:, None]
        real = i < new
        row = torch.where(real, s["cu_seqlens"][:-1, None] + i, 0)
        q = s["q"][row]
    else:
        i, new, q = torch.arange(n, device="cuda")[None], n, s["q"]
    q = q.float().view(b, n, hkv, group, D).permute(0, 2, 3, 1, 4).reshape(b, hkv, group * n, D)
    scores = torch.matmul(q, _cached(s, "k").permute(0, 2, 3, 1)).mul_(SCALE).view(b, hkv, group, n, -1)
    j = torch.arange(s["longest"], device="cuda")
    last = s["seq_lens"][:, None] - 1 + (i - new + 1 if s["causal"] else torch.zeros_like(i))  # the last key that a row sees
    scores.masked_fill_((j > last[:, None, None, :, None]), -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, hkv, group * n, -1), _cached(s, "v").transpose(1, 2)).view(b, hkv, group, n, D)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(b, n, hq, D).to(torch.bfloat16)
    lse = (top + total.log()).view(b, hq, n)
    if s["ragged"]:
        return o[real], lse.transpose(1, 2)[real].T.contiguous()
    return o, lse


# -- states --------------------------------------------------------------------------------------------------------------
def _rows(gen, *shape):
    """Keys, values or queries: N(0, 1) * 0.5, some channels of each head larger than others, as projections give them."""
    x = torch.randn(*shape, generator=gen, device="cuda", dtype=torch.bfloat16)
    channel = torch.randn(*shape[-2:], generator=gen, device="cuda").mul_(0.5).exp_().mul_(0.5)
    return x.mul_(channel)


def prepare(case, seed):
    s = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    b, hkv, page = s["batch"], s["hkv"], s["page"]
    keys, new = _lengths(case)
    s["seq_lens"] = torch.tensor(keys, dtype=torch.int32, device="cuda")
    s["cu_seqlens"] = torch.tensor([0] + [sum(new[:i + 1]) for i in range(b)], dtype=torch.int32, device="cuda")
    s["tokens"] = sum(new)
    # pages lie in any order, and some belong to nobody
    per_seq = -(-s["longest"] // page)
    needed = [-(-k // page) for k in keys]
    pages = sum(needed) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    s["page_table"] = torch.zeros(b, per_seq, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(needed):
        s["page_table"][i, :n] = order[at:at + n]
        at += n
    for which in ("k", "v"):
        x = _rows(gen, pages, page, hkv, D)
        if s["fp8"]:
            codes, scales = [], []
            for part in x.split(max(1, (64 << 20) // (page * hkv * D))):
                c, e = _quantise(part)
                codes.append(c.view(torch.uint8))
                scales.append(e)
            s[which] = torch.cat(codes).view(torch.float8_e4m3fn)
            s[which + "_scale"] = torch.cat(scales).transpose(1, 2).contiguous()  # [pages, heads, page, D / 32]
        else:
            s[which] = x
    if s["kind"] == "write":
        s["new_k"], s["new_v"] = (_rows(gen, s["tokens"], hkv, D) for _ in range(2))
    elif s["kind"] == "read":
        s["out"] = torch.zeros(2, b, s["longest"], hkv, D, dtype=torch.bfloat16, device="cuda")
    elif s["ragged"]:
        s["q"] = _rows(gen, s["tokens"], s["hq"], D)
    else:
        s["q"] = _rows(gen, b, s["most"], s["hq"], D)
    if own:
        import mercury_artifact_b200 as mb

        s["cache"] = mb.PagedKV(s["k"], s["v"], s.get("k_scale"), s.get("v_scale"))
    return s


def run(s):
    if own:
        return _run_own(s)
    return {"write": _write_plain, "read": _read_plain, "attend": _attend_plain}[s["kind"]](s)


def _run_own(s):
    import mercury_artifact_b200 as mb

    if s["kind"] == "write":
        mb.kv_cache_write(s["cache"], s["new_k"], s["new_v"], s["page_table"], s["seq_lens"], cu_seqlens=s["cu_seqlens"])
        return _cache_of(s)
    if s["kind"] == "read":
        return mb.kv_cache_read(s["cache"], s["page_table"], s["seq_lens"], out=s["out"])
    if s["ragged"]:
        return mb.attn_fwd_paged(s["q"], s["cache"], s["page_table"], s["seq_lens"], SCALE, causal=s["causal"],
                                 cu_seqlens=s["cu_seqlens"], max_queries=s["most"], max_keys=s["longest"])
    return mb.attn_fwd_paged(s["q"], s["cache"], s["page_table"], s["seq_lens"], SCALE, causal=s["causal"], max_keys=s["longest"])


# -- the definition in 64 bits -------------------------------------------------------------------------------------------
def _exact_values(s, which, i, length):
    """Cached rows [length, hkv, D] of sequence i, in 64 bits."""
    page = s["page"]
    ids = s["page_table"][i, :-(-length // page)].long()
    codes = s[which][ids].double()  # [pages, page, heads, D]
    if s["fp8"]:
        e = s[which + "_scale"][ids].double() - 127  # [pages, heads, page, D / 32]
        codes = codes * torch.exp2(e).permute(0, 2, 1, 3).repeat_interleave(BLOCK, dim=3)
    return codes.flatten(0, 1)[:length]


def _e4m3_grid():
    """The values that e4m3 holds, ascending: 0, subnormals of step 2^-9, then 3 fraction bits up to 448."""
    small = [i * 2.0 ** -9 for i in range(8)]
    return torch.tensor(small + [(1 + f / 8) * 2.0 ** e for e in range(-6, 9) for f in range(8) if (e, f) != (8, 7)],
                        dtype=torch.float64, device="cuda")


def _exact_codes(x):
    """(code values, scale bytes) of rows [T, heads, D]: nearest of the grid, ties to the even fraction."""
    t, h, _ = x.shape
    blocks = x.double().reshape(t, h, D // BLOCK, BLOCK)
    most = blocks.abs().max(-1).values
    e = torch.ceil(torch.log2(most.clamp_min(2.0 ** -1000) / 448.0) - 1e-9)  # 1e-9: far below what bf16 tells apart
    e = e + (most > 448.0 * torch.exp2(e)).double()
    e = torch.where(most > 0, e, torch.full_like(e, -50.0)).clamp(-50, 64)
    y = blocks / torch.exp2(e).unsqueeze(-1)
    grid = _e4m3_grid()
    # the value's own step: 2^-9 below 2^-6, else an eighth of its power of two; both sides of the tie are on the grid
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    z = (torch.round(y / step) * step).clamp(-448.0, 448.0)
    assert bool(torch.isin(z.abs().flatten()[:4096], grid).all())
    return z.reshape(t, h, D), (e + 127).to(torch.uint8)


def exact(case, seed):
    s = prepare(case, seed)
    keys, new = _lengths(case)
    if s["kind"] == "write":
        outs = []
        stored = {}
        for which in ("k", "v"):
            x = s["new_" + which]
            cache = s[which].double()
            scale = s[which + "_scale"].clone() if s["fp8"] else None
            at = 0
            for i in range(s["batch"]):
                where = torch.arange(keys[i] - new[i], keys[i], device="cuda")
                page, slot = s["page_table"][i].long()[where // s["page"]], where % s["page"]
                rows = x[at:at + new[i]]
                at += new[i]
                if s["fp8"]:
                    cache[page, slot], e = _exact_codes(rows)
                    scale[page, :, slot] = e
                else:
                    cache[page, slot] = rows.double()
            outs.append(cache)
            stored[which] = scale
        return outs + ([stored["k"], stored["v"]] if s["fp8"] else [])
    if s["kind"] == "read":
        out = s["out"].double()
        for c, which in enumerate(("k", "v")):
            for i in range(s["batch"]):
                out[c, i, :keys[i]] = _exact_values(s, which, i, keys[i])
        return out
    group = s["hq"] // s["hkv"]
    os, lses = [], []
    for i in range(s["batch"]):
        at = int(s["cu_seqlens"][i])
        q = (s["q"][at:at + new[i]] if s["ragged"] else s["q"][i]).double()
        o, lse = torch.zeros_like(q), torch.empty(s["hq"], new[i], dtype=torch.float64, device="cuda")
        k, v = (_exact_values(s, which, i, keys[i]) for which in ("k", "v"))
        unseen = None
        if s["causal"]:
            unseen = torch.arange(keys[i], device="cuda")[None] > torch.arange(keys[i] - new[i], keys[i], device="cuda")[:, None]
        for h in range(s["hq"]):
            score = q[:, h] @ k[:, h // group].T * SCALE
            if unseen is not None:
                score = score.masked_fill(unseen, -math.inf)
            lse[h] = torch.logsumexp(score, 1)
            p = torch.exp(score - lse[h][:, None])
            o[:, h] = torch.where(torch.isfinite(lse[h])[:, None], p, 0.0) @ v[:, h // group]
        os.append(o)
        lses.append(lse)
    if s["ragged"]:
        return torch.cat(os), torch.cat(lses, 1)
    return torch.stack(os), torch.stack(lses)
