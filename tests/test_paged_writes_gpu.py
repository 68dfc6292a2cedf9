"""kv_cache_write under offsets that do not fit: reported, and not a byte of the cache changes."""
import pytest
import torch

from tests.paged_cases import D, Batch

pytestmark = pytest.mark.gpu

FP8 = [False, True]


def _bytes(cache):
    return [t.contiguous().view(torch.uint8).clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale) if t is not None]


@pytest.mark.parametrize("fp8", FP8)
@pytest.mark.parametrize("n,sequences", [(1, 3), (10, 3), (400, 3), (2, 300)])
def test_damaged_offsets_store_nothing(fp8, n, sequences):
    """Ends beyond the tokens, negative ones, descending ones; few and many rows, more sequences than threads of a block."""
    import mercury_artifact_b200 as mb
    from mercury_artifact_b200._lib import MercuryB200Error

    batch = Batch([n + 200] * sequences, [n] * sequences, (2, 2), 16, fp8, seed=51)
    tensors = batch.cache_tensors()
    cache = mb.PagedKV(*(batch.on(t) for t in tensors))
    table, lens, tokens = batch.on(batch.table), batch.on(batch.seq_lens), batch.tokens
    new = torch.full((tokens, 2, D), 3.0, dtype=torch.bfloat16, device="cuda")
    before = _bytes(cache)
    last = sequences
    for at, value in [(last, tokens + 100), (last, 2 ** 31 - 1), (1, -2 ** 31), (1, -1), (0, -5), (0, -2 ** 31), (1, tokens + 1),
                      (last - 1, 0), (last, 0), (2, 2 ** 30)]:
        cu = batch.cu.clone()
        cu[at] = value
        mb.kv_cache_write(cache, new, new, table, lens, cu.cuda())
        with pytest.raises(MercuryB200Error, match="page number"):
            cache.check()
        assert all(torch.equal(a, b) for a, b in zip(before, _bytes(cache))), (at, value)
    # offsets as they should be: what the oracle holds, rewritten
    k, v = (torch.cat([batch.kv[i][c][batch.lens[i] - n:] for i in range(sequences)]) for c in range(2))
    mb.kv_cache_write(cache, k.cuda(), v.cuda(), table, lens, batch.on(batch.cu))
    cache.check()
    assert all(torch.equal(a, b) for a, b in zip(before, _bytes(cache)))


@pytest.mark.parametrize("fp8", FP8)
def test_rows_before_the_first_and_behind_the_last_sequence(fp8):
    """Offsets that begin above zero and end below the tokens are in order: the rows outside are nobody's."""
    import mercury_artifact_b200 as mb

    batch = Batch([60, 0, 33], [5, 0, 7], (2, 2), 16, fp8, seed=52)
    cache = mb.PagedKV(*(batch.on(t) for t in batch.cache_tensors()))
    before = _bytes(cache)
    rows = torch.full((2, 3 + batch.tokens + 4, 2, D), 9.0, dtype=torch.bfloat16)
    for c in range(2):
        rows[c, 3:3 + batch.tokens] = torch.cat([batch.kv[i][c][batch.lens[i] - m:] for i, m in enumerate(batch.new)])
    for t in (cache.k, cache.v):  # the new tokens' places
        for i, m in enumerate(batch.new):
            for j in range(batch.lens[i] - m, batch.lens[i]):
                t[batch.table[i, j // 16].item(), j % 16].view(torch.uint8).zero_()
    mb.kv_cache_write(cache, rows[0].cuda(), rows[1].cuda(), batch.on(batch.table), batch.on(batch.seq_lens), batch.on(batch.cu + 3))
    cache.check()
    assert all(torch.equal(a, b) for a, b in zip(before, _bytes(cache)))
