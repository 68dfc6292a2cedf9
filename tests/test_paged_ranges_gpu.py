"""Attention over an e4m3 cache whose powers of two differ: between blocks of 32 values, between keys, and against the
queries.  Every element of o has to keep the bound of its own column's mass, sum p |v|, however large other columns and
other keys are, and for every number of rows, so that the choice of the kernel does not show."""
import pytest
import torch

from tests.paged_cases import SCALE, Batch, bounds

pytestmark = pytest.mark.gpu

# query and K/V heads, new tokens: 1, 4, 8, 16, 32 rows a sequence and K/V head, and 40 (tiles)
ROWS = [((1, 1), 1), ((8, 2), 1), ((8, 1), 1), ((8, 2), 4), ((8, 4), 16), ((8, 2), 10)]
LENS = [[700, 90], [5003, 33, 2000]]  # units of one SM, and units that several share


def run(batch, tensors=None):
    """o within 2^-8 (half a step of bf16) for the probabilities and for the result, relative to the mass of its own element,
    and 5 % of that for the sums (tests/helpers.py: rounding_bound, without its constant); 2^-134, half of bf16's least step.
    Probabilities in f16 are rounded by 2^-11 down to 2^-24 of the largest; the scores here lie within e^16 = 2^23 of
    each other, or so far below that what they add is less than the bound."""
    import mercury_artifact_b200 as mb

    tensors = tensors or batch.cache_tensors()
    cache = mb.PagedKV(*(batch.on(t) for t in tensors))
    got_o, got_lse = mb.attn_fwd_paged(batch.on(batch.shaped(batch.q)), cache, batch.on(batch.table), batch.on(batch.seq_lens), SCALE)
    cache.check()
    o, lse, mass, size = batch.expected(tensors, True)
    got_o, got_lse = got_o.double().cpu().reshape(o.shape), got_lse.double().cpu().permute(1, 0, 2).reshape(lse.shape)
    none = torch.isinf(lse)
    assert torch.isfinite(got_o).all() and torch.equal(got_lse == -torch.inf, none)
    assert ((got_lse - lse)[~none].abs() <= bounds(o, mass, size)[1][~none]).all()
    over = (got_o - o).abs() / (1.05 * 2.0 ** -8 * (mass + o.abs()) + 2.0 ** -134)
    assert over.max().item() <= 1, f"an element of o is off by {over.max().item():.3g} times its bound"


def powers(exponents):
    """[128]: a power of two per block of 32 columns."""
    return torch.exp2(torch.tensor(exponents, dtype=torch.float64)).repeat_interleave(32)


def times(x, factor):
    return (x.double() * factor).to(torch.bfloat16)


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("heads,new", ROWS)
@pytest.mark.parametrize("exponents", [(0, -8, -12, -15), (0, -16, -24, -30), (-25, 0, -40, -50), (60, 20, -30, 0)])
def test_value_blocks_of_unequal_size(lens, heads, new, exponents):
    batch = Batch(lens, [new] * len(lens), heads, 16, True, ragged=False, seed=61, spread=2.0)
    for kv in batch.kv:
        kv[1] = times(kv[1], powers(exponents))
    run(batch)


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("heads,new", ROWS)
@pytest.mark.parametrize("low,high", [(-12, 0), (-20, 6), (-45, 60)])
def test_values_of_unequal_size(lens, heads, new, low, high):
    """Every block of every key has a power of two of its own; growing along the keys, and falling."""
    for seed in (62, 63):
        batch = Batch(lens, [new] * len(lens), heads, 16, True, ragged=False, seed=seed)
        g = torch.Generator().manual_seed(seed)
        for kv in batch.kv:
            n, h = kv.shape[1:3]
            e = torch.randint(low, high + 1, (n, h, 4), generator=g).sort(0, descending=seed == 63).values
            kv[1] = times(kv[1], torch.exp2(e.double()).repeat_interleave(32, -1))
        run(batch)


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("heads,new", ROWS)
@pytest.mark.parametrize("at", [0, 31, 64, 89, -1])
@pytest.mark.parametrize("size", [8, 14, 20, 24, 26, 40])
def test_one_large_value_block(lens, heads, new, at, size):
    """One block of one key is 2^size times the others: seen by all rows with an ordinary score, or (the last key of a causal
    call) hidden from all but the last token."""
    batch = Batch(lens, [new] * len(lens), heads, 16, True, ragged=False, seed=64)
    for i, kv in enumerate(batch.kv):
        j = min(at, kv.shape[1] - 1)
        kv[1, j, :, 32:64] = times(kv[1, j, :, 32:64], 2.0 ** size)
    run(batch)


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("heads,new", ROWS)
@pytest.mark.parametrize("at,size", [(3, 10), (3, 30), (3, 55), (70, 30), (70, 55)])
def test_a_large_value_with_a_small_score(lens, heads, new, at, size):
    """A key whose score lies 36 below the others': it counts where its values are large enough, and harms no others."""
    batch = Batch(lens, [new] * len(lens), heads, 16, True, ragged=False, seed=65)
    batch.q[..., 0] = 4.0
    for kv in batch.kv:
        kv[0, :, :, 0] = 0
        j = min(at, kv.shape[1] - 1 - new)
        kv[0, j, :, 0] = -104.0
        kv[1, j] = times(kv[1, j], 2.0 ** size)
    run(batch)


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("heads,new", ROWS)
@pytest.mark.parametrize("order", ["growing", "falling", "there and back", "in turns"])
@pytest.mark.parametrize("most", [20, 50])
def test_values_grow_as_probabilities_fall(lens, heads, new, order, most):
    """A key's value is 2^e, its probability 2^-e of the largest: every key counts alike in o."""
    batch = Batch(lens, [new] * len(lens), heads, 16, True, ragged=False, seed=71, spread=0.1)
    batch.q[..., 0] = 4.0
    for kv in batch.kv:
        n = kv.shape[1]
        j = torch.arange(n, dtype=torch.float64) / max(n - 1, 1)
        e = {"growing": j, "falling": 1 - j, "there and back": 1 - (2 * j - 1).abs(), "in turns": (torch.arange(n) // 700 % 2).double()}[order]
        e = (e * most).round()[:, None]
        kv[0, :, :, 0] = (-e * 0.6931 / (4.0 * SCALE)).to(torch.bfloat16)  # (e4m3 makes of it what it can: within 2^(e / 16))
        kv[1] = times(kv[1], torch.exp2(e)[..., None])
    run(batch)


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("heads,new", ROWS)
@pytest.mark.parametrize("exponents", [(0, 6, -9, 3), (0, 15, -15, 0), (0, 20, 5, -10), (0, 28, 14, 2)])
def test_key_blocks_of_unequal_size(lens, heads, new, exponents):
    """Keys are large where the queries are small, so that every block counts alike in the scores."""
    batch = Batch(lens, [new] * len(lens), heads, 16, True, ragged=False, seed=66, spread=2.0)
    batch.q = times(batch.q, 1 / powers(exponents))
    for kv in batch.kv:
        kv[0] = times(kv[0], powers(exponents))
    run(batch)


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("heads,new", ROWS)
@pytest.mark.parametrize("size", [12, 18, 24, 40])
def test_keys_that_are_large_where_the_queries_are_zero(lens, heads, new, size):
    """One block of some keys is 2^size times the others, and no query looks there."""
    batch = Batch(lens, [new] * len(lens), heads, 16, True, ragged=False, seed=67, spread=2.0)
    batch.q[..., 64:96] = 0
    for kv in batch.kv:
        kv[0, ::5, :, 64:96] = times(kv[0, ::5, :, 64:96], 2.0 ** size)
    run(batch)


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("heads,new", ROWS)
def test_zero_values_and_keys(lens, heads, new):
    """Blocks of zeros get the least power of two; beside others they change nothing."""
    batch = Batch(lens, [new] * len(lens), heads, 16, True, ragged=False, seed=68)
    for kv in batch.kv:
        kv[1, ::3] = 0
        kv[1, 1::3, :, :32] = 0
        kv[0, ::4] = 0
        kv[:, :40] = 0
    run(batch)


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("heads,new", ROWS)
def test_powers_of_two_that_no_write_makes(lens, heads, new):
    """Scale bytes from 3 to 76, which the cache of another program may hold."""
    batch = Batch(lens, [new] * len(lens), heads, 16, True, ragged=False, seed=69)
    g = torch.Generator().manual_seed(70)
    for lo, hi in ((60, 76), (30, 45), (3, 76)):
        k, v, ks, vs = batch.cache_tensors()
        used = vs != 255
        vs = torch.where(used, torch.randint(lo, hi + 1, vs.shape, generator=g, dtype=torch.uint8), vs)
        ks = torch.where(used, torch.randint(max(lo, 30), hi + 1, ks.shape, generator=g, dtype=torch.uint8), ks)
        run(batch, (k, v, ks, vs))


def test_every_code_under_every_scale_byte_is_read_back():
    """The code times its power of two to the nearest bf16: exact from byte 3 on; NaN from byte 192 on and for NaN codes."""
    import mercury_artifact_b200 as mb
    from oracle import paged as oracle

    cache = mb.PagedKV.empty(16, 16, 2, torch.float8_e4m3fn)
    codes = torch.arange(256, dtype=torch.uint8).view(1, 1, 2, 128).expand(16, 16, 2, 128)
    scales = torch.arange(256, dtype=torch.uint8).view(16, 1, 16, 1).expand(16, 2, 16, 4)  # a byte a slot
    for t, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        t.view(torch.uint8).copy_(codes)
        s.copy_(scales)
    table = torch.arange(16, dtype=torch.int32, device="cuda").view(1, 16)
    got = mb.kv_cache_read(cache, table, torch.tensor([256], dtype=torch.int32, device="cuda"))[:, 0].cpu()
    cache.check()
    flat = torch.arange(256, dtype=torch.uint8).view(1, 2, 128).expand(256, 2, 128)
    want = oracle.values(flat, torch.arange(256, dtype=torch.uint8).view(256, 1, 1).expand(256, 2, 4))
    want = torch.where((flat & 127) == 127, torch.full_like(want, torch.nan), want)
    assert torch.equal(want[3:192].to(torch.bfloat16).double()[~torch.isnan(want[3:192])], want[3:192][~torch.isnan(want[3:192])])
    for c in range(2):
        assert torch.equal(torch.isnan(got[c]), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got[c].float()), torch.nan_to_num(want.to(torch.bfloat16).float()))
