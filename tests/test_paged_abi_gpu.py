"""The paged calls through the C ABI, where a caller chooses bounds and workspace itself."""
import pytest
import torch

from tests.paged_cases import D, SCALE, Batch, check

pytestmark = pytest.mark.gpu

FP8 = [False, True]


def attend(batch, cache, max_queries, max_keys=None, causal=True, table=None, fill=None):
    """o, lse of mb_attn_paged in buffers that held 7; the workspace holds bytes of `fill`."""
    from mercury_artifact_b200 import _lib

    ragged = batch.ragged
    q = batch.on(batch.shaped(batch.q))
    b, n = len(batch.lens), batch.new[0]
    cu = batch.on(batch.cu) if ragged else None
    table = batch.on(batch.table) if table is None else table
    lens = batch.on(batch.seq_lens)
    o = torch.full_like(q, 7.0)
    lse = torch.full((batch.hq, batch.tokens) if ragged else (b, batch.hq, n), 7.0, device="cuda")
    rows = (0, batch.hq * D, D) if ragged else (n * batch.hq * D, batch.hq * D, D)
    args = _lib.ATTN_PAGED.pack(
        *cache._batch(table, lens, cu, batch.tokens), q.data_ptr(), *rows, o.data_ptr(), *rows, lse.data_ptr(),
        0 if ragged else batch.hq * n, batch.tokens if ragged else n, batch.hq, max_queries,
        table.shape[1] * batch.page_size if max_keys is None else max_keys, int(causal), SCALE)
    need = _lib.lib.mb_attn_paged_workspace(args)
    ws = torch.full((max(need, 1),), 0 if fill is None else fill, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    _lib.check(_lib.lib.mb_attn_paged(args, ws.data_ptr() if need else None, need, stream), "mb_attn_paged")
    return o, lse


def make(batch):
    import mercury_artifact_b200 as mb

    tensors = batch.cache_tensors()
    return tensors, mb.PagedKV(*(batch.on(t) for t in tensors))


@pytest.mark.parametrize("fp8", FP8)
@pytest.mark.parametrize("heads", [(8, 2), (8, 8), (32, 1)])
@pytest.mark.parametrize("n,bound", [(1, 1), (1, 2), (1, 64), (2, 5), (3, 300), (5, 2 ** 30), (40, 41), (40, 1000)])
def test_bound_above_the_new_tokens_of_a_padded_batch(fp8, heads, n, bound):
    """max_queries is an upper bound: every row is written, whichever kernel the bound alone would have chosen."""
    batch = Batch([700, 1, 130, 0, 2 * n], [n] * 5, heads, 16, fp8, ragged=False, seed=41)
    tensors, cache = make(batch)
    o, lse = attend(batch, cache, bound)
    cache.check()
    check(batch, o, lse, batch.expected(tensors, True))


@pytest.mark.parametrize("fp8", FP8)
@pytest.mark.parametrize("new,known", [([0, 0], True), ([1, 0], False), ([0, 40], False)])
def test_bound_of_no_new_tokens(fp8, new, known):
    """max_queries = 0 of a ragged batch: nothing to write, or a report."""
    from mercury_artifact_b200._lib import MercuryB200Error

    batch = Batch([100, 50], new, (8, 2), 16, fp8, seed=42)
    _, cache = make(batch)
    if known:  # rows behind the last sequence
        batch.q, batch.tokens = torch.zeros(3, 8, D, dtype=torch.bfloat16), 3
    o, lse = attend(batch, cache, 0)
    if known:
        cache.check()
    else:
        with pytest.raises(MercuryB200Error, match="page number"):
            cache.check()
    assert (o == 7).all() and (lse == 7).all()


@pytest.mark.parametrize("fp8", FP8)
@pytest.mark.parametrize("page", [16, 24, 7])
@pytest.mark.parametrize("new", [1, 5, 40, 100])
def test_keys_of_a_bad_page_are_zeros(fp8, page, new):
    """Every path puts zeros where a page number is bad, whatever the workspace held: results are finite and repeat."""
    from mercury_artifact_b200._lib import MercuryB200Error

    batch = Batch([130, 260, 100], [new] * 3, (8, 2), page, fp8, ragged=False, seed=43)
    tensors, cache = make(batch)
    good = batch.table.clone()
    used = {int(x) for i, n in enumerate(batch.lens) for x in good[i, :-(-n // page)]}
    zeros = next(p for p in range(batch.pages) if p not in used)
    for t, value in zip(tensors, (0, 0, 127, 127)):
        if t is not None:
            t[zeros].view(torch.uint8).fill_(value)
    batch.table[1, 2] = zeros
    want = batch.expected(tensors, True)
    bad = good.clone()
    bad[1, 2] = batch.pages + 3
    results = [attend(batch, cache, new, table=bad.cuda(), fill=fill) for fill in (0, 0xff, 0x7f)]
    with pytest.raises(MercuryB200Error, match="page number"):
        cache.check()
    for o, lse in results:
        check(batch, o, lse, want)
        assert torch.equal(o, results[0][0]) and torch.equal(lse, results[0][1])


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,new,covered", [([300, 700, 64, 129, 1000], [40, 100, 64, 33, 257], 131072),  # two sequences a group
                                              ([300, 0, 700, 500, 64, 200, 90], [40, 0, 1, 3, 64, 0, 90], 131072),  # single tokens too
                                              ([700, 40, 1300], [90, 40, 100], 300000)])  # one sequence a group
def test_chunks_of_a_quantised_cache_in_groups(causal, lens, new, covered):
    """A bound on the keys so high that the bf16 copy of all sequences would not fit: group by group, in the same memory.
    The copy starts as NaN."""
    batch = Batch(lens, new, (16, 8), 16, True, seed=44)
    tensors, cache = make(batch)
    want = batch.expected(tensors, causal)
    table = torch.full((len(lens), covered // 16), 2 ** 30, dtype=torch.int32, device="cuda")
    table[:, :batch.table.shape[1]] = batch.on(batch.table)
    assert len(lens) * covered * 8 * 512 > 1 << 30
    results = [attend(batch, cache, max(new), causal=causal, table=table, fill=0xff) for _ in range(2)]
    cache.check()
    for o, lse in results:
        check(batch, o, lse, want)
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])


@pytest.mark.parametrize("fp8", FP8)
@pytest.mark.parametrize("new", [1, 40, 300])
def test_cache_whose_heads_are_one(fp8, new):
    """A view that repeats one head: read, and attended to by few and by many rows, like its copy."""
    import mercury_artifact_b200 as mb

    batch = Batch([500, 300], [new, new], (8, 2), 16, fp8, ragged=False, seed=45)
    for kv in batch.kv:
        kv[:, :, 1] = kv[:, :, 0]
    k, v, ks, vs = batch.cache_tensors()
    want = batch.expected((k, v, ks, vs), True)
    one = torch.stack([k.view(torch.uint8), v.view(torch.uint8)])[:, :, :, :1].contiguous().cuda().view(k.dtype)
    cache = mb.PagedKV(one[0].expand(-1, -1, 2, -1), one[1].expand(-1, -1, 2, -1), batch.on(ks), batch.on(vs))
    assert cache.k.stride(2) == 0
    o, lse = attend(batch, cache, new)
    cache.check()
    check(batch, o, lse, want)
    kv = mb.kv_cache_read(cache, batch.on(batch.table), batch.on(batch.seq_lens), max_keys=300)
    assert torch.equal(kv[:, 1, :, 0], kv[:, 1, :, 1]) and not torch.isnan(kv).any()
