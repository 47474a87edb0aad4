"""What the C entry points of the 8-bit KV cache refuse on the host, before any CUDA call."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def native():
    from flash_attn_triton_b200.build import build
    build()
    from flash_attn_triton_b200 import _native as N
    return N


def cache(N, **kw):
    c = N.Cache8()
    c.code, c.block, c.k_scale, c.v_scale = 0, 16, 4096, 4096
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def decode(N, **kw):
    d = N.DecodeArgs()
    d.heads_q, d.heads_kv, d.head_dim, d.batch, d.seqlen_q, d.page_size, d.num_pages = 8, 2, 128, 1, 1, 64, 4
    d.q = d.o = d.k_cache = d.v_cache = d.cache_seqlens = 4096       # never dereferenced
    for f in ("q_stride", "o_stride", "kc_stride", "vc_stride"):
        setattr(d, f, N._I64x3(1024, 1024, 128))
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_decode(native):
    N, lib = native, native.lib()
    failed = ctypes.c_uint32()
    for d, c, word in ((decode(N), cache(N, code=2), "code"), (decode(N), cache(N, block=0), "1 to 1024"), (decode(N), cache(N, block=1025), "1 to 1024"),
                       (decode(N), cache(N, block=48), "multiple of the scale block"), (decode(N), cache(N, k_scale=None), "scales are required"),
                       (decode(N, k_cache=4096 + 8), cache(N), "16-byte"), (decode(N, kc_stride=N._I64x3(1024, 1024, 120)), cache(N), "16-byte"),
                       (decode(N, head_dim=96), cache(N), "head dimension"), (decode(N, page_size=0), cache(N), "page_size"),
                       (decode(N), None, "cache is NULL"), (decode(N), cache(N), "workspace")):
        ptr = None if c is None else ctypes.byref(c)
        for got in (lib.fa_decode_paged8(ctypes.byref(d), ptr, None), lib.fa_decode_paged8_checked(ctypes.byref(d), ptr, ctypes.byref(failed), None)):
            assert got < 0
            if word != "workspace":                                  # (that needs the device first)
                assert got == -1 and word in lib.fa_last_error().decode(), lib.fa_last_error()
    assert lib.fa_decode_paged8(None, None, None) == -1
    assert lib.fa_decode_paged8_checked(ctypes.byref(decode(N)), ctypes.byref(cache(N)), None, None) == -1
    assert lib.fa_decode8_workspace_bytes(None, None) == 0 and lib.fa_decode8_counters(None, None) == 0
    assert lib.fa_decode8_workspace_bytes(ctypes.byref(decode(N, batch=0)), ctypes.byref(cache(N))) == 0
    assert lib.fa_decode8_counters(ctypes.byref(decode(N)), ctypes.byref(cache(N))) >= 0


def append(N, **kw):
    a = N.Append8Args()
    a.heads, a.head_dim, a.tokens, a.page_size, a.num_pages, a.cache = 2, 128, 5, 64, 4, cache(N)
    a.k = a.v = a.k_cache = a.v_cache = a.slots = 4096
    a.k_stride = a.v_stride = (ctypes.c_int64 * 2)(256, 128)
    a.kc_stride = a.vc_stride = N._I64x3(1024, 1024, 128)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_append(native):
    N, lib = native, native.lib()
    failed = ctypes.c_uint32()
    for a, word in ((append(N, dtype=2), "dtype"), (append(N, head_dim=48), "head dimension"), (append(N, tokens=-1), "size"), (append(N, heads=0), "size"),
                    (append(N, tokens=2 ** 31), "size"), (append(N, slots=None), "required"), (append(N, k=4098), "16-byte"),
                    (append(N, v_stride=(ctypes.c_int64 * 2)(256, 124)), "16-byte"), (append(N, cache=cache(N, block=7)), "multiple of the scale block"),
                    (append(N, cache=cache(N, code=5)), "code"), (append(N, workspace=4), "workspace"), (append(N, num_pages=-1), "size")):
        for got in (lib.fa_append8(ctypes.byref(a), None), lib.fa_append8_checked(ctypes.byref(a), ctypes.byref(failed), None)):
            assert got == -1 and word in lib.fa_last_error().decode(), lib.fa_last_error()
    assert lib.fa_append8(None, None) == -1
    assert lib.fa_append8_workspace_bytes(ctypes.byref(append(N))) >= 4 * 4 // 8
    assert lib.fa_append8_workspace_bytes(ctypes.byref(append(N, tokens=0))) == 0 and lib.fa_append8_workspace_bytes(None) == 0


def table(N, **kw):
    a = N.BlockTableArgs()
    a.batch, a.page_size, a.num_free, a.table_pages, a.table_stride, a.num_slots = 2, 16, 4, 4, 4, 8
    for f in ("cache_seqlens", "new_lens", "free_pages", "block_table", "slots", "cu_seqlens", "pages_used"):
        setattr(a, f, 4096)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_block_table(native):
    N, lib = native, native.lib()
    failed = ctypes.c_uint32()
    for a, word in ((table(N, batch=-1), "negative"), (table(N, num_slots=2 ** 31), "too many"), (table(N, num_free=2 ** 31), "too many"),
                    (table(N, page_size=0), "page_size"), (table(N, slots=None), "required"), (table(N, new_lens=None), "required"),
                    (table(N, block_table=None), "required"), (table(N, free_pages=None), "required")):
        for got in (lib.fa_block_table(ctypes.byref(a), None), lib.fa_block_table_checked(ctypes.byref(a), ctypes.byref(failed), None)):
            assert got == -1 and word in lib.fa_last_error().decode(), lib.fa_last_error()
    assert lib.fa_block_table(None, None) == -1


def test_public_calls_refuse_cpu_tensors():
    import torch
    import flash_attn_triton as fa
    q, c, s = torch.zeros(1, 1, 2, 64, dtype=torch.float16), torch.zeros(2, 16, 2, 64, dtype=torch.int8), torch.zeros(2, 1, 2)
    n = torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        fa.flash_attn_with_kvcache(q, c, c, cache_seqlens=n, k_scale=s, v_scale=s)
    with pytest.raises(ValueError, match="CUDA"):
        fa.kvcache_append(q[0], q[0], c, c, n, s, s)
    with pytest.raises(ValueError, match="CUDA"):
        fa.build_block_table(n, n, n, torch.zeros(1, 2, dtype=torch.int32), 16, 1)
