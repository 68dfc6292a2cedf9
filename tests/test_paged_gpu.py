"""Keys and values in pages on the GPU, against plain 64-bit code (oracle/paged.py)."""
import pytest
import torch

from oracle import paged as oracle
from tests.paged_cases import D, SCALE, Batch, check

pytestmark = pytest.mark.gpu

FP8 = [False, True]


def _mb():
    import mercury_artifact_b200 as mb

    return mb


def _cache(batch, tensors):
    return _mb().PagedKV(*(batch.on(t) for t in tensors))


def _status():
    from mercury_artifact_b200 import _lib

    return _lib.status_fetch(torch.cuda.current_stream().cuda_stream)


def _attend(batch, cache, causal=True, **more):
    if batch.ragged:
        more.setdefault("cu_seqlens", batch.on(batch.cu))
        more.setdefault("max_queries", max(batch.new + [0]))
    return _mb().attn_fwd_paged(batch.on(batch.shaped(batch.q)), cache, batch.on(batch.table), batch.on(batch.seq_lens), SCALE,
                                causal=causal, **more)


# -- writing and reading -----------------------------------------------------------------------------------------------
WRITES = [
    # lens, new, hkv, page_size
    ([1], [1], 1, 16),
    ([5, 0, 33], [5, 0, 33], 2, 16),
    ([100, 17, 1, 64], [1, 1, 1, 1], 8, 16),
    ([300, 129, 7], [200, 128, 7], 3, 24),
    ([50, 50], [50, 50], 4, 1),
    ([1000, 3], [999, 1], 8, 64),
    ([70, 70, 70], [70, 70, 70], 5, 7),
]


@pytest.mark.parametrize("fp8", FP8)
@pytest.mark.parametrize("lens,new,hkv,page", WRITES)
def test_write_then_read(fp8, lens, new, hkv, page):
    """Every slot of the cache holds what the oracle's does, bit for bit, also those that are not written."""
    batch = Batch(lens, new, (hkv, hkv), page, fp8, seed=3)
    before = batch.cache_tensors()
    for i, n in enumerate(new):  # new values for the new tokens
        batch.kv[i][:, lens[i] - n:] *= -1.75
    after = batch.cache_tensors()
    cache = _cache(batch, before)
    k, v = (torch.cat([batch.kv[i][c][lens[i] - n:] for i, n in enumerate(new)]) for c in range(2))
    _mb().kv_cache_write(cache, batch.on(k), batch.on(v), batch.on(batch.table), batch.on(batch.seq_lens), batch.on(batch.cu))
    for got, want in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), after):
        if want is not None:
            kind = torch.uint8 if fp8 else torch.int16
            assert torch.equal(got.cpu().view(kind), want.view(kind))
    out = torch.full((2, len(lens), max(lens) + 3, hkv, D), 7.0, dtype=torch.bfloat16, device="cuda")
    assert _mb().kv_cache_read(cache, batch.on(batch.table), batch.on(batch.seq_lens), out=out) is out
    assert _status() == 0
    for i, n in enumerate(lens):
        for c in range(2):
            want = oracle.gather(after[c], after[2 + c], batch.table[i], n, page)
            assert torch.equal(out[c, i, :n].double().cpu(), want)
        assert (out[:, i, n:] == 7).all()
    short = _mb().kv_cache_read(cache, batch.on(batch.table), batch.on(batch.seq_lens), max_keys=2)
    for i, n in enumerate(lens):
        assert torch.equal(short[:, i, :min(n, 2)], out[:, i, :min(n, 2)]) and (short[:, i, min(n, 2):] == 0).all()


def test_write_padded_batch_strided_rows():
    """[batch, n, heads, D] new tokens that are views, more tokens than keys in one sequence."""
    batch = Batch([40, 2, 9], [4, 4, 4], (2, 2), 16, True, seed=5)
    want = batch.cache_tensors()
    cache = _cache(batch, want)
    cache.k.view(torch.uint8).fill_(1)
    cache.v.view(torch.uint8).fill_(1)
    cache.k_scale.fill_(99)
    cache.v_scale.fill_(99)
    rows = torch.zeros(2, 3, 4, 2, D, dtype=torch.bfloat16)
    for i, n in enumerate(batch.lens):
        have = min(n, 4)
        rows[:, i, 4 - have:] = batch.kv[i][:, n - have:]
    wide = torch.zeros(2, 3, 4, 5, D + 8, dtype=torch.bfloat16, device="cuda")
    wide[:, :, :, 1:3, :D] = rows.cuda()
    _mb().kv_cache_write(cache, wide[0, :, :, 1:3, :D], wide[1, :, :, 1:3, :D], batch.on(batch.table), batch.on(batch.seq_lens))
    assert _status() == 0
    written = 0
    for i, n in enumerate(batch.lens):
        for j in range(max(0, n - 4), n):
            page, slot = batch.table[i, j // 16].item(), j % 16
            for got, w in ((cache.k, want[0]), (cache.v, want[1])):
                assert torch.equal(got[page, slot].cpu().view(torch.uint8), w[page, slot].view(torch.uint8))
            for got, w in ((cache.k_scale, want[2]), (cache.v_scale, want[3])):
                assert torch.equal(got[page, :, slot].cpu(), w[page, :, slot])
            written += 1
    assert (cache.k_scale != 99).sum().item() <= written * 2 * 4  # and nothing else
    assert (cache.k.view(torch.uint8) != 1).any(-1).sum().item() <= written * 2


def test_quantising_edges():
    """Ties, subnormal codes, the exponent's limits, zeros of both signs, infinities and NaN."""
    top = 448.0
    blocks = [
        [top], [top * 1.0078125], [top / 2], [1.0625 * 2.0 ** k for k in range(-6, 9)], [1.1875, 1.3125, -1.0625, top],
        [2.0 ** -9 * k / 2 for k in range(16)] + [top], [-0.0, 0.0], [2.0 ** -60, 2.0 ** -59], [2.0 ** -50, 3 * 2.0 ** -52],
        [2.0 ** 72, 2.0 ** 73, -(2.0 ** 75)], [3.3e38, -3.3e38], [1e-40, 2.0 ** -126], [2.0 ** 120, 1.0],
        [float("inf"), 1.0], [float("nan"), 2.0], [float("-inf")],
    ]
    x = torch.zeros(len(blocks), 1, D, dtype=torch.bfloat16)
    for i, b in enumerate(blocks):
        x[i, 0, 32 * (i % 4):32 * (i % 4) + len(b)] = torch.tensor(b, dtype=torch.float64).to(torch.bfloat16)
    n = len(blocks)
    cache = _mb().PagedKV.empty(2, 16, 1, torch.float8_e4m3fn)
    table, lens = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda"), torch.tensor([n], dtype=torch.int32, device="cuda")
    _mb().kv_cache_write(cache, x[None].cuda(), -x[None].cuda(), table, lens)
    got = _mb().kv_cache_read(cache, table, lens, max_keys=n)[:, 0].cpu()
    codes, scales = oracle.quantise(x)
    for c, sign in ((0, 1), (1, -1)):
        want = oracle.values(codes, scales) * sign
        assert torch.equal(torch.isnan(got[c]), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got[c].double()), torch.nan_to_num(want))
    bytes_ = torch.cat([cache.k_scale[1, 0], cache.k_scale[0, 0]])[:n].cpu()
    assert torch.equal(bytes_, scales[:, 0])


# -- attention ---------------------------------------------------------------------------------------------------------
HEADS = [(1, 1), (8, 8), (8, 2), (14, 2), (16, 1), (32, 8), (32, 1)]


@pytest.mark.parametrize("fp8", FP8)
@pytest.mark.parametrize("heads", HEADS)
def test_one_token(fp8, heads):
    """Lengths around the ends of pages and steps, an empty sequence among them."""
    batch = Batch([1, 15, 16, 17, 0, 127, 128, 129, 255, 257, 700], [1] * 11, heads, 16, fp8, ragged=False, seed=1)
    tensors = batch.cache_tensors()
    o, lse = _attend(batch, _cache(batch, tensors))
    assert _status() == 0
    check(batch, o, lse, batch.expected(tensors, True))


@pytest.mark.parametrize("fp8", FP8)
@pytest.mark.parametrize("page", [1, 7, 16, 24, 64, 128, 1000])
def test_page_sizes(fp8, page):
    batch = Batch([513, 90, 1200], [2, 1, 3], (8, 2), page, fp8, seed=2)
    tensors = batch.cache_tensors()
    o, lse = _attend(batch, _cache(batch, tensors))
    assert _status() == 0
    check(batch, o, lse, batch.expected(tensors, True))


@pytest.mark.parametrize("fp8", FP8)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new", [2, 3, 5, 8])
def test_few_tokens(fp8, causal, new):
    """Drafted tokens: rows of one sequence see different numbers of keys; some see none."""
    batch = Batch([new - 1, new, 100, 128 + new, 3000, 1], [new] * 6, (8, 2), 16, fp8, ragged=False, seed=4, spread=2.0)
    tensors = batch.cache_tensors()
    o, lse = _attend(batch, _cache(batch, tensors), causal)
    assert _status() == 0
    check(batch, o, lse, batch.expected(tensors, causal))


@pytest.mark.parametrize("fp8", FP8)
def test_one_long_sequence_over_all_sms(fp8):
    """One sequence, one K/V head: its keys are split over every SM and merged; and bits repeat."""
    batch = Batch([70001], [1], (4, 1), 64, fp8, ragged=False, seed=6, spread=2.0)
    tensors = batch.cache_tensors()
    cache = _cache(batch, tensors)
    o, lse = _attend(batch, cache)
    o2, lse2 = _attend(batch, cache)
    assert _status() == 0
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    o_, lse_, mass, size = batch.expected(tensors, True)
    check(batch, o, lse, (o_, lse_, mass, size))


@pytest.mark.parametrize("fp8", FP8)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads", [(1, 1), (8, 8), (8, 2), (14, 2), (16, 1)])
def test_chunks_ragged(fp8, causal, heads):
    """Chunks around the sizes of tiles beside single tokens and nothing: both kernels in one call."""
    lens = [1, 64, 300, 128, 129, 0, 257, 1000, 40, 5]
    new = [1, 64, 7, 128, 127, 0, 257, 33, 90, 0]  # the ninth has more new tokens than keys
    batch = Batch(lens, new, heads, 16, fp8, seed=7, spread=2.0)
    tensors = batch.cache_tensors()
    o, lse = _attend(batch, _cache(batch, tensors), causal)
    assert _status() == 0
    check(batch, o, lse, batch.expected(tensors, causal))


@pytest.mark.parametrize("fp8", FP8)
@pytest.mark.parametrize("page", [1, 7, 24, 128, 1000])
def test_chunks_page_sizes(fp8, page):
    batch = Batch([513, 90, 1200], [100, 90, 270], (8, 2), page, fp8, seed=8)
    tensors = batch.cache_tensors()
    o, lse = _attend(batch, _cache(batch, tensors))
    assert _status() == 0
    check(batch, o, lse, batch.expected(tensors, True))


@pytest.mark.parametrize("fp8", FP8)
@pytest.mark.parametrize("lens,new,heads", [([5000], [64], (8, 2)), ([4000, 100], [150, 150], (4, 4)), ([3000], [1500], (2, 1)),
                                            ([20000], [40], (4, 4))])
def test_chunks_split_over_keys(fp8, lens, new, heads):
    """Few units against many keys: shares and their merge; bits repeat."""
    batch = Batch(lens, new, heads, 64, fp8, ragged=False, seed=9, spread=2.0)
    tensors = batch.cache_tensors()
    cache = _cache(batch, tensors)
    o, lse = _attend(batch, cache)
    o2, lse2 = _attend(batch, cache)
    assert _status() == 0
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    check(batch, o, lse, batch.expected(tensors, True))
