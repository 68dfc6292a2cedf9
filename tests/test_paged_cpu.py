"""Paged K/V cache without a GPU: refusals, argument blocks, and the oracle against torch's own e4m3."""
import ctypes as C
import math
import re
import subprocess
from pathlib import Path

import pytest
import torch

from oracle import paged as oracle

ROOT = Path(__file__).resolve().parent.parent


def test_oracle_rounds_like_torch():
    x = torch.cat([torch.linspace(-500, 500, 20001), torch.randn(20000) * 2, torch.randn(20000) * 2.0 ** -8,
                   torch.tensor([k * 2.0 ** -10 for k in range(-40, 41)])]).clamp(-448, 448)
    codes = oracle.nearest_e4m3(x)
    want = x.to(torch.float8_e4m3fn)
    assert torch.equal(codes, want.view(torch.uint8))
    assert torch.equal(oracle.code_values(codes), want.double())


@pytest.mark.parametrize("size", [2.0 ** -70, 2.0 ** -52, 1e-3, 1.0, 448.0, 1e9, 2.0 ** 71, 3e38])
def test_scale_is_the_least_power_of_two(size):
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(50, 2, 128, generator=g).clamp(-1, 1) * size).to(torch.bfloat16)
    codes, scales = oracle.quantise(x)
    e = scales.double() - 127
    most = x.double().unflatten(-1, (4, 32)).abs().amax(-1)
    assert ((most <= 448 * torch.exp2(e)) | (e == 64)).all()
    assert ((most > 448 * torch.exp2(e - 1)) | (e == -50)).all()
    back = oracle.values(codes, scales)
    inside = (most <= 448 * torch.exp2(e)).unsqueeze(-1)
    off = (back - x.double()).abs().unflatten(-1, (4, 32))
    # half a step: 2^-4 of the value, or half of the least step 2^-9 of the block
    assert (off <= torch.maximum(x.double().abs().unflatten(-1, (4, 32)) * 2.0 ** -4, torch.exp2(e - 10).unsqueeze(-1)))[inside.expand_as(off)].all()
    assert torch.equal(back, back.to(torch.bfloat16).double())  # exact in bf16


def test_argument_blocks_have_the_layout_of_the_header(tmp_path):
    from mercury_artifact_b200 import _lib

    source = tmp_path / "sizes.c"
    fields = {"mb_paged_kv": _lib.PagedKVArgs, "mb_attn_paged_args": _lib.AttnPagedArgs}
    lines = [f'printf("%zu ", sizeof({name}));' for name in fields]
    lines += [f'printf("%zu ", offsetof({name}, {f}));' for name, s in fields.items() for f, _ in s._fields_]
    source.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "mercury_b200.h"\nint main(void) {' + "".join(lines) + "return 0;}\n")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(source), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = [C.sizeof(s) for s in fields.values()] + [getattr(s, f).offset for s in fields.values() for f, _ in s._fields_]
    assert got == want
    assert _lib.PAGED_KV.size == got[0] and _lib.ATTN_PAGED.size == got[1]
    values = list(range(1, len(re.sub("0P$", "", _lib.ATTN_PAGED.format)[1:]) + 1))
    block = _lib.AttnPagedArgs.from_buffer_copy(_lib.ATTN_PAGED.pack(*values))
    assert block.kv.k == 1 and block.kv.status == 20 and block.q == 21 and block.softmax_scale == values[-1]


def _kv(_lib, **changes):
    a = _lib.PagedKVArgs()
    a.k = a.v = a.page_table = a.seq_lens = 1 << 20
    a.stride_page, a.stride_slot, a.stride_h = 16 * 2 * 128, 2 * 128, 128
    a.batch, a.tokens, a.pages, a.page_size, a.max_pages, a.hkv, a.head_dim, a.dtype = 1, 1, 4, 16, 4, 2, 128, 0
    for name, value in changes.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("changes,code", [
    (dict(head_dim=64), -2), (dict(dtype=1), -2), (dict(page_size=0), -1), (dict(batch=-1), -1), (dict(hkv=0), -1), (dict(k=None), -1),
    (dict(k=(1 << 20) + 8), -1), (dict(stride_slot=2 * 128 + 4), -1), (dict(seq_lens=None), -1), (dict(page_table=None), -1),
    (dict(max_pages=2 ** 30), -1), (dict(batch=2, tokens=3), -1), (dict(dtype=2), -1),
    (dict(dtype=2, k_scale=1 << 20, v_scale=(1 << 20) + 2), -1),
])
def test_library_refuses_bad_caches(changes, code):
    from mercury_artifact_b200 import _lib

    a = _kv(_lib, **changes)
    assert _lib.lib.mb_kv_cache_write(C.byref(a), 1 << 20, 1 << 20, 0, 256, 128, None) == code
    assert _lib.lib.mb_kv_cache_read(C.byref(a), 1 << 20, 1 << 20, 0, 256, 128, 4, None) == code
    q = _lib.AttnPagedArgs()
    q.kv = a
    q.q = q.o = q.lse = 1 << 20
    q.hq, q.max_queries, q.max_keys, q.softmax_scale = 4, 1, 64, 1.0
    assert _lib.lib.mb_attn_paged(C.byref(q), None, 0, None) == code


def test_library_refuses_null_blocks():
    from mercury_artifact_b200 import _lib

    assert _lib.lib.mb_kv_cache_write(None, None, None, 0, 0, 0, None) == -1
    assert _lib.lib.mb_kv_cache_read(None, None, None, 0, 0, 0, 0, None) == -1
    assert _lib.lib.mb_attn_paged(None, None, 0, None) == -1
    assert _lib.lib.mb_attn_paged_workspace(None) == 0


def _pages(dtype=torch.bfloat16, *shape):
    return torch.zeros(*(shape or (4, 16, 2, 128)), dtype=torch.uint8).to(dtype) if dtype != torch.float8_e4m3fn else \
        torch.zeros(*(shape or (4, 16, 2, 128)), dtype=torch.uint8).view(dtype)


def test_cache_refusals():
    import mercury_artifact_b200 as mb

    k = _pages()
    for bad, error, match in [
        (lambda: mb.PagedKV(k[0], k[0]), ValueError, "page_size"),
        (lambda: mb.PagedKV(k.float(), k.float()), TypeError, "bfloat16"),
        (lambda: mb.PagedKV(k, k[:3]), ValueError, "share"),
        (lambda: mb.PagedKV(_pages(torch.bfloat16, 4, 16, 2, 64), _pages(torch.bfloat16, 4, 16, 2, 64)), NotImplementedError, "head_dim"),
        (lambda: mb.PagedKV(k.transpose(2, 3), k.transpose(2, 3)), NotImplementedError, "head_dim"),
        (lambda: mb.PagedKV(_pages(torch.bfloat16, 4, 16, 2, 132)[..., :128], _pages(torch.bfloat16, 4, 16, 2, 132)[..., :128]), ValueError, "16 bytes"),
        (lambda: mb.PagedKV(k, k, torch.zeros(1, dtype=torch.uint8), None), ValueError, "scales"),
        (lambda: mb.PagedKV(_pages(torch.float8_e4m3fn), _pages(torch.float8_e4m3fn)), ValueError, "k_scale"),
        (lambda: mb.PagedKV(_pages(torch.float8_e4m3fn), _pages(torch.float8_e4m3fn), torch.zeros(4, 2, 16, 4), torch.zeros(4, 2, 16, 4)), ValueError, "k_scale"),
        (lambda: mb.PagedKV(k, k), ValueError, "CUDA"),
    ]:
        with pytest.raises(error, match=match):
            bad()


class _CpuCache:
    """What the call wrappers look at, on the CPU: their refusals come before anything is launched."""

    def __new__(cls):
        import mercury_artifact_b200 as mb

        cache = object.__new__(mb.PagedKV)
        cache.device, cache.dtype = torch.device("cpu"), torch.bfloat16
        cache.pages, cache.page_size, cache.heads = 4, 16, 2
        cache._head, cache._tail, cache._kind = (0,) * 7, (4, 16), (2, 128, 0, 0)
        return cache


def test_call_refusals():
    import mercury_artifact_b200 as mb

    cache = _CpuCache()
    table, lens = torch.zeros(3, 4, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    cu = torch.tensor([0, 1, 2, 4], dtype=torch.int32)

    def rows(*shape, dtype=torch.bfloat16):
        return torch.zeros(*shape, 128, dtype=dtype)

    q, k = rows(3, 1, 4), rows(3, 1, 2)
    attend = [
        ((rows(3, 1, 3), table, lens, 1.0), {}, "multiple"),
        ((rows(3, 4), table, lens, 1.0), {}, "must be"),
        ((q, table, lens, 0.0), {}, "softmax_scale"),
        ((q, table, lens, math.nan), {}, "softmax_scale"),
        ((q, table, lens, math.inf), {}, "softmax_scale"),
        ((q, table.long(), lens, 1.0), {}, "page_table"),
        ((q, table[0], lens, 1.0), {}, "page_table|batch"),
        ((q, table.T, lens, 1.0), {}, "page_table|batch"),
        ((q, table, lens.long(), 1.0), {}, "seq_lens"),
        ((q, table, lens[:2], 1.0), {}, "seq_lens"),
        ((q, table[:2], lens[:2], 1.0), {}, "batch"),
        ((q, table, lens, 1.0), {"max_queries": 0}, "max_queries"),
        ((q, table, lens, 1.0), {"max_keys": -1}, "max_keys"),
        ((q, table, lens, 1.0), {"out": rows(3, 1, 5)}, "out"),
        ((q, table, lens, 1.0), {"lse": torch.zeros(3, 1, 4)}, "lse"),
        ((q, table, lens, 1.0), {"lse": torch.zeros(3, 4, 1, dtype=torch.float64)}, "lse"),
        ((rows(4, 4), table, lens, 1.0), {"cu_seqlens": cu.long()}, "cu_seqlens"),
        ((rows(4, 4), table, lens, 1.0), {"cu_seqlens": cu[:3]}, "cu_seqlens"),
        ((q, table, lens, 1.0), {"cu_seqlens": cu}, "must be"),
    ]
    for args, kw, match in attend:
        with pytest.raises(ValueError, match=match):
            mb.attn_fwd_paged(args[0], cache, *args[1:], **kw)
    with pytest.raises(TypeError):
        mb.attn_fwd_paged(rows(3, 1, 4, dtype=torch.float16), cache, table, lens, 1.0)
    with pytest.raises(ValueError, match="16 bytes"):
        mb.attn_fwd_paged(torch.zeros(3, 1, 4, 132, dtype=torch.bfloat16)[..., :128], cache, table, lens, 1.0)
    for args, match in [((k, rows(3, 2, 2)), "share"), ((rows(3, 1, 4), rows(3, 1, 4)), "heads"), ((rows(2, 1, 2), rows(2, 1, 2)), "batch"),
                        ((rows(3, 2), rows(3, 2)), "must be")]:
        with pytest.raises(ValueError, match=match):
            mb.kv_cache_write(cache, *args, table, lens)
    for kw, match in [({"out": rows(2, 3, 4, 3)}, "out"), ({"out": rows(2, 2, 4, 2)}, "out"), ({"out": rows(2, 3, 4, 2), "max_keys": 5}, "max_keys"),
                      ({"max_keys": -1}, "max_keys")]:
        with pytest.raises(ValueError, match=match):
            mb.kv_cache_read(cache, table, lens, **kw)


def test_status_of_a_failed_check_has_its_own_words():
    from mercury_artifact_b200 import _lib

    assert "check failed" in _lib._status_text(110, "device-side timeout") and "page number" in _lib._status_text(110, "")
    assert _lib._status_text(109, "device-side timeout").startswith("device-side timeout: ")
