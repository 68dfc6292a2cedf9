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
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,new", [((8, 2), 1), ((8, 2), 2), ((8, 2), 3), ((8, 2), 8), ((12, 6), 5), ((3, 3), 7), ((6, 3), 2),
                                       ((14, 2), 1), ((14, 2), 2), ((4, 4), 32)])
def test_few_tokens_split_over_sms(fp8, causal, heads, new):
    """Units that several SMs share, of an even and an odd number of K/V heads, in one block of rows and in more; bits repeat."""
    batch = Batch([5000, 4097, new, 129 + new, 700], [new] * 5, heads, 16, fp8, ragged=False, seed=24, spread=2.0)
    tensors = batch.cache_tensors()
    cache = _cache(batch, tensors)
    o, lse = _attend(batch, cache, causal)
    o2, lse2 = _attend(batch, cache, causal)
    assert _status() == 0
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    check(batch, o, lse, batch.expected(tensors, causal))


@pytest.mark.parametrize("page", [8, 32, 40, 64, 96])
def test_chunks_box_sizes(page):
    """Every way a tile of keys is cut into boxes of pages."""
    batch = Batch([page, 127, 129, 1000, 385], [page, 127, 100, 64, 385], (8, 2), page, seed=25)
    tensors = batch.cache_tensors()
    o, lse = _attend(batch, _cache(batch, tensors))
    assert _status() == 0
    check(batch, o, lse, batch.expected(tensors, True))


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


# -- what calls may find -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fp8", FP8)
@pytest.mark.parametrize("new", [[1, 3, 2], [40, 1, 90]])
def test_rows_behind_the_last_sequence_and_given_buffers(fp8, new):
    """q, out and lse are views of wider buffers with rows behind the last sequence; these stay as they were."""
    batch = Batch([200, 31, 300], new, (8, 2), 16, fp8, seed=11)
    tensors = batch.cache_tensors()
    t = batch.tokens
    wide = torch.full((t + 7, 10, D + 8), 3.0, dtype=torch.bfloat16, device="cuda")
    wide[:t, 1:9, :D] = batch.q.cuda()
    out = torch.full((t + 7, 9, D), 5.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((8, t + 20), 6.0, device="cuda")
    o, l = _mb().attn_fwd_paged(wide[:, 1:9, :D], _cache(batch, tensors), batch.on(batch.table), batch.on(batch.seq_lens), SCALE,
                                cu_seqlens=batch.on(batch.cu), max_queries=max(new), out=out[:, :8], lse=lse[:, 3:3 + t + 7])
    assert _status() == 0
    check(batch, o[:t], l[:, :t], batch.expected(tensors, True))
    assert (out[t:] == 5).all() and (out[:, 8] == 5).all()
    assert (lse[:, :3] == 6).all() and (lse[:, 3 + t:] == 6).all()


@pytest.mark.parametrize("fp8", FP8)
@pytest.mark.parametrize("new", [1, 60])
def test_cache_layouts(fp8, new):
    """Heads before slots, and keys and values as the halves of one packed tensor with pages between them unused."""
    batch = Batch([333, 70], [new, new], (8, 4), 16, fp8, ragged=False, seed=12)
    k, v, ks, vs = batch.cache_tensors()
    want = batch.expected((k, v, ks, vs), True)
    bits = torch.uint8 if fp8 else torch.int16
    shape = (2, batch.pages * 2, 4, 16, D)  # every other page, heads first
    packed = torch.zeros(shape, dtype=bits, device="cuda")
    packed[0, ::2], packed[1, ::2] = (x.view(bits).transpose(1, 2).cuda() for x in (k, v))
    packed = packed.view(k.dtype)[:, ::2].transpose(2, 3)
    cache = _mb().PagedKV(packed[0], packed[1], batch.on(ks), batch.on(vs))
    o, lse = _attend(batch, cache)
    assert _status() == 0
    check(batch, o, lse, want)
    back = _mb().kv_cache_read(cache, batch.on(batch.table), batch.on(batch.seq_lens), max_keys=333)
    for c, (x, s) in enumerate(((k, ks), (v, vs))):
        assert torch.equal(back[c, 0].double().cpu(), oracle.gather(x, s, batch.table[0], 333, 16))


@pytest.mark.parametrize("fp8", FP8)
@pytest.mark.parametrize("sequences", [300, 1100])
def test_many_sequences(fp8, sequences):
    """More sequences than threads of a block, some of them empty, some without new tokens."""
    lens = [(7 * i) % 61 for i in range(sequences)]
    new = [min(n, (i % 4)) for i, n in enumerate(lens)]
    new[5], lens[5] = 30, 40  # one chunk for the tiles
    batch = Batch(lens, new, (4, 1), 16, fp8, seed=13)
    tensors = batch.cache_tensors()
    cache = _cache(batch, tensors)
    o, lse = _attend(batch, cache)
    assert _status() == 0
    check(batch, o, lse, batch.expected(tensors, True))
    k, v = (torch.cat([batch.kv[i][c][lens[i] - n:] for i, n in enumerate(new)]) for c in range(2))
    cache.k.view(torch.uint8).zero_()
    _mb().kv_cache_write(cache, batch.on(k), batch.on(v), batch.on(batch.table), batch.on(batch.seq_lens), batch.on(batch.cu))
    assert _status() == 0
    for i in (0, 5, 63, 255, 256, 257, sequences - 1):
        for j in range(lens[i] - new[i], lens[i]):
            page, slot = batch.table[i, j // 16].item(), j % 16
            assert torch.equal(cache.k[page, slot].cpu().view(torch.uint8), tensors[0][page, slot].view(torch.uint8))


def test_offsets_beyond_32_bits():
    """Pages whose addresses lie more than 2^32 bytes (and 2^31 elements) behind the cache's."""
    pages, page, heads = 300000, 16, 8
    need = 2 * pages * page * heads * D * 2
    if torch.cuda.mem_get_info()[0] < need + (8 << 30):
        pytest.skip("needs 20 GB of device memory")
    cache = _mb().PagedKV.empty(pages, page, heads)
    g = torch.Generator().manual_seed(0)
    for new in (1, 40):
        k, v, q = ((torch.randn(2, 100, heads, D, generator=g)).to(torch.bfloat16) for _ in range(3))
        q = q[:, :new]
        table = torch.tensor([[pages - 1 - i for i in range(7)], [pages // 2 + 131 * i for i in range(7)]], dtype=torch.int32, device="cuda")
        lens = torch.tensor([100, 100], dtype=torch.int32, device="cuda")
        _mb().kv_cache_write(cache, k.cuda(), v.cuda(), table, lens)
        o, lse = _mb().attn_fwd_paged(q.cuda(), cache, table, lens, SCALE)
        back = _mb().kv_cache_read(cache, table, lens, max_keys=100)
        assert _status() == 0
        assert torch.equal(back[0].cpu(), k) and torch.equal(back[1].cpu(), v)
        from tests.paged_cases import bounds

        for b in range(2):
            want, l, mass, size = oracle.attend(q[b], k[b].double(), v[b].double(), SCALE, True)
            tol, tol_l = bounds(want, mass, size)
            assert ((o[b].double().cpu() - want).abs() <= tol).all()
            assert ((lse[b].double().cpu() - l).abs() <= tol_l).all()


def test_empty_calls():
    mb = _mb()
    cache = mb.PagedKV.empty(4, 16, 2)
    table = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")

    def rows(*shape):
        return torch.zeros(*shape, D, dtype=torch.bfloat16, device="cuda")

    o, lse = mb.attn_fwd_paged(rows(3, 0, 4), cache, table, lens, SCALE)
    assert o.shape == (3, 0, 4, D) and lse.shape == (3, 4, 0)
    o, lse = mb.attn_fwd_paged(rows(0, 2, 4), cache, table[:0], lens[:0], SCALE)
    assert o.shape == (0, 2, 4, D)
    for n in (1, 40):  # nothing cached, by length, by bound, and by a table without columns
        for kw in ({}, {"max_keys": 0}):
            o, lse = mb.attn_fwd_paged(rows(3, n, 4) + 1, cache, table, lens, SCALE, **kw)
            assert (o == 0).all() and (lse == float("-inf")).all()
        o, lse = mb.attn_fwd_paged(rows(3, n, 4) + 1, cache, table[:, :0], lens, SCALE)
        assert (o == 0).all() and (lse == float("-inf")).all()
    mb.kv_cache_write(cache, rows(3, 0, 2), rows(3, 0, 2), table, lens)
    mb.kv_cache_write(cache, rows(3, 2, 2), rows(3, 2, 2), table, lens)  # more new tokens than keys: none is stored
    assert mb.kv_cache_read(cache, table, lens, max_keys=0).shape == (2, 3, 0, 2, D)
    assert (mb.kv_cache_read(cache, table, lens) == 0).all()
    none = mb.PagedKV.empty(0, 16, 2)
    o, lse = mb.attn_fwd_paged(rows(3, 40, 4), none, table, lens, SCALE)
    assert (lse == float("-inf")).all()
    assert _status() == 0


@pytest.mark.parametrize("fp8", FP8)
@pytest.mark.parametrize("new", [1, 5, 50])
def test_bad_pages_lengths_and_offsets_are_reported(fp8, new):
    """What lies outside is skipped and reported; the other sequences and the next call are as they should be."""
    from mercury_artifact_b200._lib import MercuryB200Error

    mb = _mb()
    batch = Batch([100, 120, 90], [new] * 3, (8, 2), 16, fp8, seed=14)
    tensors = batch.cache_tensors()
    cache = _cache(batch, tensors)
    want = batch.expected(tensors, True)
    q, cu = batch.on(batch.q), batch.on(batch.cu)
    table, lens = batch.on(batch.table), batch.on(batch.seq_lens)
    new_rows = torch.zeros(batch.tokens, 2, D, dtype=torch.bfloat16, device="cuda")

    def damaged(t, at, value):
        t = t.clone()
        t[at] = value
        return t

    cases = [(damaged(table, (1, 3), batch.pages), lens, cu), (damaged(table, (1, 0), -1), lens, cu),
             (table, damaged(lens, 1, -5), cu), (table, damaged(lens, 1, 2 ** 30), cu),
             (table, lens, damaged(cu, 3, batch.tokens + 100)), (table, lens, damaged(cu, 1, -2 ** 31))]
    for tb, ln, c in cases:
        o, lse = mb.attn_fwd_paged(q, cache, tb, ln, SCALE, cu_seqlens=c, max_queries=new)
        with pytest.raises(MercuryB200Error, match="page number"):
            cache.check()
        if c is cu:  # the sequences beside the damaged one
            for i in (0, 2):
                rows = slice(int(batch.cu[i]), int(batch.cu[i + 1]))
                err = (o[rows].double().cpu() - want[0][rows]).abs().max().item()
                assert err < 0.05
        if new == 1:
            mb.kv_cache_read(cache, tb, ln, max_keys=128)
            if c is cu:
                with pytest.raises(MercuryB200Error):
                    cache.check()
    # a write does not leave the pages
    before = cache.k.view(torch.uint8).clone()
    mb.kv_cache_write(cache, new_rows, new_rows, torch.full_like(table, batch.pages), lens, cu)
    with pytest.raises(MercuryB200Error):
        cache.check()
    assert torch.equal(before, cache.k.view(torch.uint8))
    o, lse = mb.attn_fwd_paged(q, cache, table, lens, SCALE, cu_seqlens=cu, max_queries=new)
    cache.check()
    check(batch, o, lse, want)


@pytest.mark.parametrize("fp8", [False, True])
def test_offsets_that_ask_for_more_work_than_a_launch_has(fp8):
    """Offsets that do not ascend give every other sequence all tokens: more units, each split over several SMs, than the
    launch was cut for.  It is reported, and nothing but o and lse is written."""
    from mercury_artifact_b200._lib import MercuryB200Error

    mb = _mb()
    batch = Batch([4096] * 6, [256] + [0] * 5, (8, 1), 16, fp8, seed=21)
    cache = _cache(batch, batch.cache_tensors())
    cu = torch.tensor([0, 256, 0, 256, 0, 256, 0], dtype=torch.int32, device="cuda")
    guard = torch.full((300, 8, D), 7.0, dtype=torch.bfloat16, device="cuda")
    for _ in range(2):
        mb.attn_fwd_paged(batch.on(batch.q), cache, batch.on(batch.table), batch.on(batch.seq_lens), SCALE, cu_seqlens=cu,
                          out=guard[:256])
        with pytest.raises(MercuryB200Error, match="page number"):
            cache.check()
    assert (guard[256:] == 7).all()
    o, lse = mb.attn_fwd_paged(batch.on(batch.q), cache, batch.on(batch.table), batch.on(batch.seq_lens), SCALE,
                               cu_seqlens=batch.on(batch.cu))
    cache.check()
    check(batch, o, lse, batch.expected(batch.cache_tensors(), True))


def test_more_sequences_than_a_grid_dimension_has():
    """70 000 sequences of at most one key share a page."""
    mb = _mb()
    n = 70000
    cache = mb.PagedKV.empty(1, 16, 1)
    g = torch.Generator().manual_seed(22)
    rows = torch.randn(2, 16, 1, D, generator=g).to(torch.bfloat16).cuda()
    cache.k[0], cache.v[0] = rows[0], rows[1]
    table = torch.zeros(n, 1, dtype=torch.int32, device="cuda")
    lens = (torch.arange(n, device="cuda") % 2).to(torch.int32)
    got = mb.kv_cache_read(cache, table, lens, max_keys=1)
    want = rows[:, None, :1] * lens.view(1, n, 1, 1, 1)
    assert torch.equal(got, want.to(torch.bfloat16))
    q = torch.randn(n, 1, 1, D, generator=g).to(torch.bfloat16).cuda()
    o, lse = mb.attn_fwd_paged(q, cache, table, lens, SCALE)
    cache.check()
    assert torch.equal(o[1::2], rows[1, :1].expand(n // 2, 1, 1, D)) and (o[0::2] == 0).all()
    assert torch.isinf(lse[0::2]).all() and torch.isfinite(lse[1::2]).all()


@pytest.mark.parametrize("fp8", FP8)
@pytest.mark.parametrize("new", [1, 5, 100])
def test_bound_of_no_keys(fp8, new):
    """max_keys=0: rows that see nothing; a sequence that has keys is reported."""
    from mercury_artifact_b200._lib import MercuryB200Error

    mb = _mb()
    batch = Batch([0, 0], [new] * 2, (8, 2), 16, fp8, ragged=False, seed=26)
    tensors = batch.cache_tensors()
    o, lse = _attend(batch, _cache(batch, tensors), max_keys=0)
    assert _status() == 0
    check(batch, o, lse, batch.expected(tensors, True))
    batch = Batch([0, 9], [new] * 2, (8, 2), 16, fp8, ragged=False, seed=27)
    cache = _cache(batch, batch.cache_tensors())
    _attend(batch, cache, max_keys=0)
    with pytest.raises(MercuryB200Error, match="page number"):
        cache.check()


def test_bound_of_no_new_tokens():
    """max_queries=0: right where no sequence has any, reported where one has more than a token."""
    from mercury_artifact_b200._lib import MercuryB200Error

    mb = _mb()
    batch = Batch([40, 50], [5, 2], (4, 2), 16, seed=23)
    cache = _cache(batch, batch.cache_tensors())
    q, table, lens = batch.on(batch.q), batch.on(batch.table), batch.on(batch.seq_lens)
    out = torch.full_like(q, 7.0)
    none = torch.zeros(3, dtype=torch.int32, device="cuda")
    mb.attn_fwd_paged(q, cache, table, lens, SCALE, cu_seqlens=none, max_queries=0, out=out)
    cache.check()
    assert (out == 7).all()
    mb.attn_fwd_paged(q, cache, table, lens, SCALE, cu_seqlens=batch.on(batch.cu), max_queries=0)
    with pytest.raises(MercuryB200Error, match="page number"):
        cache.check()


@pytest.mark.parametrize("fp8", FP8)
def test_captured_graph_replays_with_other_lengths(fp8):
    """Write, attend and attend with a chunk, captured once; the lengths, pages and rows change between replays."""
    mb = _mb()
    a = Batch([100, 0, 517], [1, 1, 1], (8, 2), 16, fp8, ragged=False, seed=15)
    b = Batch([17, 600, 33], [1, 1, 1], (8, 2), 16, fp8, ragged=False, seed=16)
    pages = max(a.pages, b.pages)
    cache = mb.PagedKV.empty(pages, 16, 2, torch.float8_e4m3fn if fp8 else torch.bfloat16)
    table = torch.zeros(3, 40, dtype=torch.int32, device="cuda")
    lens = torch.ones(3, dtype=torch.int32, device="cuda")
    q = torch.zeros(3, 1, 8, D, dtype=torch.bfloat16, device="cuda")
    kv = torch.zeros(2, 3, 1, 2, D, dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm up
        mb.kv_cache_write(cache, kv[0], kv[1], table, lens)
        mb.attn_fwd_paged(q, cache, table, lens, SCALE)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mb.kv_cache_write(cache, kv[0], kv[1], table, lens)
        o, lse = mb.attn_fwd_paged(q, cache, table, lens, SCALE)
        o2, lse2 = mb.attn_fwd_paged(q, cache, table, lens, SCALE, max_keys=640)
    for batch in (a, b, a):
        tensors = batch.cache_tensors()
        for got, x in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), tensors):
            if x is not None:
                got[:batch.pages].view(torch.uint8).copy_(x.view(torch.uint8))
        table[:, :batch.table.shape[1]] = batch.on(batch.table)
        lens.copy_(batch.seq_lens)
        q.copy_(batch.shaped(batch.q))
        for i, n in enumerate(batch.lens):  # the last key arrives with the call
            if n:
                kv[:, i, 0] = batch.kv[i][:, n - 1].cuda()
                cache.k[batch.table[i, (n - 1) // 16].item(), (n - 1) % 16].view(torch.uint8).fill_(0x7f)
        graph.replay()
        cache.check()
        want = batch.expected(tensors, True)
        check(batch, o, lse, want)
        check(batch, o2, lse2, want)


def test_two_streams_at_once():
    """Calls on two streams, each with scratch of its own, give what they give alone."""
    mb = _mb()
    work = []
    for seed, fp8, lens, new in ((17, False, [9000], [1]), (18, True, [9000], [1]), (19, False, [5000], [40]), (20, True, [700, 9000], [9, 9])):
        batch = Batch(lens, new, (4, 1), 16, fp8, ragged=False, seed=seed)
        cache = _cache(batch, batch.cache_tensors())
        args = (batch.on(batch.shaped(batch.q)), cache, batch.on(batch.table), batch.on(batch.seq_lens), SCALE)
        work.append((args, mb.attn_fwd_paged(*args)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    results = [[] for _ in work]
    for _ in range(20):
        for (args, _), stream, got in zip(work, streams, results):
            with torch.cuda.stream(stream):
                got.append(mb.attn_fwd_paged(*args))
    torch.cuda.synchronize()
    for (_, want), got in zip(work, results):
        for o, lse in got:
            assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
    assert _status() == 0


@pytest.mark.parametrize("fp8", FP8)
@pytest.mark.parametrize("lens,new,heads,page", [([3000], [100], (8, 2), 64), ([3000] * 4, [100] * 4, (8, 8), 16), ([500] * 3, [300] * 3, (8, 8), 7),
                                                 ([2000] * 9, [3] * 9, (8, 2), 16)])
def test_bits_repeat(fp8, lens, new, heads, page):
    """With caches cold and warm: every value that is used was waited for."""
    batch = Batch(lens, new, heads, page, fp8, ragged=False, seed=21)
    cache = _cache(batch, batch.cache_tensors())
    args = (batch.on(batch.shaped(batch.q)), cache, batch.on(batch.table), batch.on(batch.seq_lens), SCALE)
    flush = torch.empty(64 << 20, dtype=torch.int32, device="cuda")
    runs = []
    for i in range(40):
        if i % 4 == 0:
            flush.fill_(i)
        runs.append(_mb().attn_fwd_paged(*args))
        if i % 3 == 0:
            torch.cuda.synchronize()
    assert _status() == 0
    for o, lse in runs[1:]:
        assert torch.equal(o, runs[0][0]) and torch.equal(lse, runs[0][1])


# -- values ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("new", [1, 6, 40])
@pytest.mark.parametrize("k_size,v_size", [(1.0, 2.0 ** -40), (1.0, 2.0 ** 60), (2.0 ** -20, 1.0), (2.0 ** 12, 2.0 ** -12)])
def test_magnitudes_of_a_quantised_cache(new, k_size, v_size):
    """Keys and values far from one: the powers of two go into the scores' scale and the results, not into f16's range."""
    batch = Batch([400, 129], [new, new], (8, 2), 16, True, ragged=False, seed=22, spread=0.5 / max(k_size, 1.0))
    for kv in batch.kv:
        kv[0] *= k_size
        kv[1] *= v_size
    tensors = batch.cache_tensors()
    o, lse = _attend(batch, _cache(batch, tensors))
    assert _status() == 0
    o_, lse_, mass, size = batch.expected(tensors, True)
    check(batch, o.double() / v_size, lse, (o_ / v_size, lse_, mass / v_size, size))


@pytest.mark.parametrize("new", [1, 40])
def test_blocks_that_are_not_numbers(new):
    """A key or value block with a NaN makes the rows that see it NaN; sequences that do not hold it stay."""
    for which in (0, 1):
        batch = Batch([200, 90], [new, new], (4, 1), 16, True, ragged=False, seed=23)
        batch.kv[0][which, 100, 0, 40] = float("inf")
        tensors = batch.cache_tensors()
        o, lse = _attend(batch, _cache(batch, tensors))
        assert _status() == 0
        assert torch.isnan(o[0].float()[..., 32:64]).all()
        assert torch.isnan(o[0].float()).all() == (which == 0)
        assert torch.isnan(lse[0]).all() == (which == 0)
        assert not torch.isnan(o[1].float()).any()
        second = Batch([90], [new], (4, 1), 16, True, ragged=False)
        second.lens, second.new, second.tokens = [90], [new], new
        second.table, second.seq_lens, second.q, second.cu = batch.table[1:], batch.seq_lens[1:], batch.q[new:], batch.cu[:2]
        check(second, o[1:], lse[1:], second.expected(tensors, True))


@pytest.mark.parametrize("new", [1, 8, 60])
def test_codes_that_are_not_numbers(new):
    """A NaN code in a cache that something else has written: NaN wherever it is read, by every kernel, and nowhere else."""
    for which in (0, 1):
        batch = Batch([200, 90], [new, new], (4, 2), 16, True, ragged=False, seed=28)
        tensors = batch.cache_tensors()
        want = batch.expected(tensors, True)
        cache = _cache(batch, tensors)
        page, slot = batch.table[0, 100 // 16].item(), 100 % 16
        (cache.v if which else cache.k).view(torch.uint8)[page, slot, 0, 40] = 0xff if which else 0x7f
        kv = _mb().kv_cache_read(cache, batch.on(batch.table), batch.on(batch.seq_lens), max_keys=200)
        assert torch.isnan(kv).sum().item() == 1 and torch.isnan(kv[which, 0, 100, 0, 40])
        o, lse = _attend(batch, cache)
        assert _status() == 0
        first = o[0, :, :2].float()  # the query heads of K/V head 0; every new token sees key 100
        if which:
            assert torch.isnan(first[..., 40]).all() and torch.isnan(o).sum().item() == 2 * new
            assert not torch.isnan(lse).any()
        else:
            assert torch.isnan(first).all() and torch.isnan(o).sum().item() == 2 * new * D and torch.isnan(lse).sum().item() == 2 * new
        nan = torch.isnan(o).view(-1, 4, D).cpu()
        clean = torch.where(nan, want[0].to(torch.bfloat16), o.view(-1, 4, D).cpu())
        none = torch.isnan(lse).cpu()
        clean_lse = torch.where(none, want[1].view(4, 2, new).permute(1, 0, 2).float(), lse.cpu())
        check(batch, clean, clean_lse, want)


# -- together ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fp8", FP8)
def test_serving_run(fp8):
    """A prompt in chunks, then tokens one by one: each call sees what was written before it; sequences share a prefix."""
    mb = _mb()
    g = torch.Generator().manual_seed(31)
    hq, hkv, page, total = 8, 2, 16, 150
    cache = mb.PagedKV.empty(40, page, hkv, torch.float8_e4m3fn if fp8 else torch.bfloat16)
    k, v = ((torch.randn(2, total, hkv, D, generator=g)).to(torch.bfloat16) for _ in range(2))
    q = torch.randn(2, total, hq, D, generator=g).to(torch.bfloat16)
    for x in (k, v, q):
        x[1, :64] = x[0, :64]  # the second sequence begins like the first one, in the same four pages
    table = torch.arange(20, dtype=torch.int32).reshape(2, 10)
    table[1, :4] = table[0, :4]
    table = table.cuda()
    at = [0, 64]  # the shared prefix is written once
    steps = [(64, 0), (33, 50), (1, 1), (1, 1), (3, 2), (20, 1), (1, 30)]
    for n0, n1 in steps:
        new = [n0, n1]
        at = [at[0] + n0, at[1] + n1]
        lens = torch.tensor(at, dtype=torch.int32)
        cu = torch.tensor([0, n0, n0 + n1], dtype=torch.int32, device="cuda")
        kn, vn, qn = (torch.cat([x[i, at[i] - new[i]:at[i]] for i in range(2)]).cuda() for x in (k, v, q))
        mb.kv_cache_write(cache, kn, vn, table, lens.cuda(), cu)
        o, lse = mb.attn_fwd_paged(qn, cache, table, lens.cuda(), SCALE, cu_seqlens=cu, max_queries=max(new))
        cache.check()
        row = 0
        for i in range(2):
            kk, vv = k[i, :at[i]].double(), v[i, :at[i]].double()
            if fp8:
                kk, vv = (oracle.values(*oracle.quantise(x[i, :at[i]])) for x in (k, v))
            want, l, mass, size = oracle.attend(q[i, at[i] - new[i]:at[i]], kk, vv, SCALE, True)
            from tests.paged_cases import bounds

            tol, tol_l = bounds(want, mass, size)
            got = o[row:row + new[i]].double().cpu()
            assert ((got - want).abs() <= tol).all()
            assert ((lse[:, row:row + new[i]].double().cpu() - l).abs() <= tol_l).all()
            row += new[i]


def test_cache_and_block_merge_and_ring_reads_back():
    """A cached prefix and a block of fresh keys, merged like two blocks of a ring, are attention over both; what is read back
    goes into the fused forward."""
    from oracle import block
    from mercury_artifact_b200.ring import RingAttention

    mb = _mb()
    g = torch.Generator().manual_seed(32)
    b, prefix, n, hq, hkv = 2, 300, 128, 8, 2
    k, v = ((torch.randn(b, prefix + n, hkv, D, generator=g) * 0.5).to(torch.bfloat16).cuda() for _ in range(2))
    q = (torch.randn(b, n, hq, D, generator=g) * 0.5).to(torch.bfloat16).cuda()
    cache = mb.PagedKV.empty(64, 16, hkv)
    table = torch.randperm(64, generator=g)[:b * 20].reshape(b, 20).to(torch.int32).cuda()
    lens = torch.full((b,), prefix, dtype=torch.int32, device="cuda")
    mb.kv_cache_write(cache, k[:, :prefix], v[:, :prefix], table, lens)
    o1, l1 = mb.attn_fwd_paged(q, cache, table, lens, SCALE, causal=False)
    o2, l2, _, _ = mb._flash_attn_forward(q, k[:, prefix:], v[:, prefix:], 0.0, SCALE, True)
    out, ls = mb.update_out_and_lse(None, None, o1, l1)
    out, ls = mb.update_out_and_lse(out, ls, o2, l2)
    ro, rl = block.block_attn_fwd(q.cpu(), k.cpu(), v.cpu(), SCALE, causal=True, q_off=prefix, k_off=0)
    assert (out.cpu() - ro.float()).abs().max().item() <= 2e-2
    assert (ls.squeeze(-1).permute(0, 2, 1).cpu() - rl).abs().max().item() <= 1e-3
    kv = mb.kv_cache_read(cache, table, lens, max_keys=prefix)
    op = RingAttention((1,), b, prefix, hq, hkv, D, causal=True)
    qq = torch.randn(b, prefix, hq, D, generator=g).to(torch.bfloat16).cuda()
    o3, l3 = op.forward(qq, kv)
    o4, l4 = mb.attn_fwd_paged(qq, cache, table, lens, SCALE)
    assert (o3.float() - o4.float()).abs().max().item() <= 2e-2 and (l3 - l4).abs().max().item() <= 1e-3
    assert _status() == 0
