"""What the calls around drafted trees refuse on the host: the Python calls, and the C entry points before any CUDA call."""
import ctypes

import pytest
import torch

import flash_attn_triton_b200 as fa


@pytest.fixture(scope="module")
def native():
    from flash_attn_triton_b200.build import build
    build()
    from flash_attn_triton_b200 import _native as N
    return N


def t(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype)


def ints(*shape, dtype=torch.int32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("change,match", [
    (dict(q=t(2, 64)), "shape"), (dict(k=t(2, 4, 2, 64)), "shape"), (dict(k=t(2, 5, 2, 32)), "shape"), (dict(k=t(10, 2, 64)), "shape"),
    (dict(q=t(2, 5, 4, 64).double()), "FP16"), (dict(k=t(2, 5, 2, 64, dtype=torch.bfloat16)), "matching"),
    (dict(q=t(2, 5, 4, 48), k=t(2, 5, 2, 48)), "head dimension"), (dict(k=t(2, 5, 0, 64)), "at least one head"),
    (dict(q_weight=t(32)), "weights"), (dict(q_weight=t(64, dtype=torch.bfloat16)), "weights"),
    (dict(q_weight=t(64), k_weight=t(64, dtype=torch.float32)), "weights"), (dict(rotary_cos=t(9, 8)), "together"),
    (dict(rotary_cos=t(9, 8), rotary_sin=t(9, 4)), "seqlen_ro"), (dict(rotary_cos=t(9, 40), rotary_sin=t(9, 40)), "exceed"),
    (dict(rotary_cos=t(9, 8, dtype=torch.bfloat16), rotary_sin=t(9, 8, dtype=torch.bfloat16)), "tables"),
    (dict(rotary_cos=t(9, 8, dtype=torch.float32).requires_grad_(), rotary_sin=t(9, 8, dtype=torch.float32)), "gradients"),
    (dict(positions=ints(2, 4)), "positions"), (dict(positions=t(2, 5)), "positions"), (dict(positions=ints(2, 1)), "positions"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(), "CUDA")])
def test_qk_norm_rotary(change, match):
    kw = dict(q=t(2, 5, 4, 64), k=t(2, 5, 2, 64))
    kw.update(change)
    with pytest.raises(ValueError, match=match):
        fa.qk_norm_rotary(**kw)


@pytest.mark.parametrize("change,match", [
    (dict(target_probs=t(2, 3)), "same shape"), (dict(draft_probs=t(2, 3, 8)), "same shape"), (dict(draft_probs=t(2, 3, 7, dtype=torch.float32)), "matching"),
    (dict(target_probs=t(2, 0, 7), draft_probs=t(2, 0, 7)), "1024"), (dict(target_probs=t(2, 1025, 1), draft_probs=t(2, 1025, 1)), "1024"),
    (dict(target_probs=t(2, 3, 0), draft_probs=t(2, 3, 0)), "vocabulary"), (dict(draft_tokens=t(2, 3)), "draft_tokens"),
    (dict(draft_tokens=ints(2, 4)), "draft_tokens"), (dict(parents=ints(4)), "parents"), (dict(parents=t(3)), "parents"),
    (dict(accept_uniforms=t(2, 3)), "FP32"), (dict(sample_uniforms=t(2).double()), "FP32"),
    (dict(accept_uniforms=t(2, 4, dtype=torch.float32)), "shape"), (dict(sample_uniforms=t(2, 1, dtype=torch.float32)), "shape"), (dict(), "CUDA")])
def test_verify_draft_tree(change, match):
    kw = dict(draft_tokens=ints(2, 3), parents=ints(3), target_probs=t(2, 3, 7), draft_probs=t(2, 3, 7),
              accept_uniforms=t(2, 3, dtype=torch.float32), sample_uniforms=t(2, dtype=torch.float32))
    kw.update(change)
    with pytest.raises(ValueError, match=match):
        fa.verify_draft_tree(**kw)


@pytest.mark.parametrize("change,match", [
    (dict(k_cache=[]), "tensors"), (dict(k_cache=[t(4, 16, 2, 64)] * 2), "as many"), (dict(v_cache=t(4, 16, 2, 32)), "same shape"),
    (dict(k_cache=t(4, 16, 64), v_cache=t(4, 16, 64)), "same shape"), (dict(k_cache=t(4, 16, 2, 64).float(), v_cache=t(4, 16, 2, 64).float()), "FP16"),
    (dict(k_cache=t(4, 16, 2, 48), v_cache=t(4, 16, 2, 48)), "head dimension"), (dict(k_cache=t(4, 16, 0, 64), v_cache=t(4, 16, 0, 64)), "head"),
    (dict(k_cache=[t(4, 16, 2, 64), t(4, 2, 16, 64).transpose(1, 2)], v_cache=[t(4, 16, 2, 64), t(4, 16, 2, 64)]), "strides"),
    (dict(k_cache=t(4, 16, 64, 2).transpose(2, 3)[..., :2, :], v_cache=t(4, 16, 2, 64)), "unit"),
    (dict(path=ints(2)), "path"), (dict(path=t(2, 3)), "path"), (dict(block_table=ints(3, 2)), "block_table"), (dict(block_table=t(2, 2)), "integer"),
    (dict(block_table=ints(2, 2), cache_leftpad=ints(2)), "leftpad"), (dict(block_table=ints(2, 2), cache_batch_idx=ints(2)), "batch_idx"),
    (dict(path=ints(5, 3)), "cache_batch_idx"), (dict(), "CUDA")])
def test_kvcache_compact(change, match):
    kw = dict(k_cache=t(4, 16, 2, 64), v_cache=t(4, 16, 2, 64), cache_seqlens=ints(2), path=ints(2, 3), num_accepted=ints(2))
    kw.update(change)
    with pytest.raises(ValueError, match=match):
        fa.kvcache_compact(**kw)


@pytest.mark.parametrize("change,match", [
    (dict(block_table=ints(2)), "block_table"), (dict(block_table=ints(2, 3, dtype=torch.int64)), "int32"),
    (dict(block_table=ints(3, 2).T), "unit stride"), (dict(page_size=0), "page_size"), (dict(num_pages=-1), "num_pages"),
    (dict(num_pages=2 ** 31), "num_pages"), (dict(), "CUDA")])
def test_release_pages(change, match):
    kw = dict(held_lens=ints(2), kept_lens=ints(2), block_table=ints(2, 3), page_size=16, num_pages=4)
    kw.update(change)
    with pytest.raises(ValueError, match=match):
        fa.release_pages(**kw)


def test_entry_points_refuse_before_cuda(native):
    N, lib, ref = native, native.lib(), ctypes.byref
    failed = ctypes.c_uint32()

    def err(got, word):
        assert got == -1 and word in lib.fa_last_error().decode(), (got, lib.fa_last_error())

    def verify(**kw):
        a = N.VerifyArgs()
        a.batch, a.nodes, a.vocab = 1, 4, 100
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.fa_verify_draft_tree(ref(a), None)
    err(lib.fa_verify_draft_tree(None, None), "NULL")
    for kw, word in ((dict(dtype=3), "dtype"), (dict(batch=-1), "batch"), (dict(nodes=0), "1024"), (dict(nodes=1025), "1024"),
                     (dict(vocab=0), "vocabulary"), (dict(vocab=2 ** 31), "vocabulary"), (dict(), "NULL")):
        err(verify(**kw), word)
    assert verify(batch=0) == 0

    def compact(**kw):
        a = N.CompactArgs()
        a.layers, a.batch, a.heads, a.head_dim, a.page_size, a.num_pages, a.path_len, a.path_stride = 2, 1, 2, 64, 16, 4, 3, 3
        a.k_cache = (ctypes.c_void_p * 2)(1 << 20, 2 << 20)
        a.v_cache = (ctypes.c_void_p * 2)(3 << 20, 4 << 20)
        a.kc_stride = a.vc_stride = N._I64x3(2048, 128, 64)
        a.cache_seqlens = a.path = a.num_accepted = 4096
        for k, v in kw.items():
            setattr(a, k, v)
        got = lib.fa_compact(ref(a), None), lib.fa_compact_checked(ref(a), ref(failed), None)
        assert got[0] == got[1]
        return got[0]
    err(lib.fa_compact(None, None), "NULL")
    pointers = ctypes.c_void_p * 2
    for kw, word in ((dict(layers=-1), "layers"), (dict(layers=129), "layers"), (dict(batch=-1), "size"), (dict(head_dim=96), "head dimension"),
                     (dict(page_size=0), "page_size"), (dict(block_table=4096), "block_table_stride"), (dict(path=None), "NULL"),
                     (dict(block_table=4096, block_table_stride=1, cache_leftpad=4096), "leftpad"), (dict(kc_stride=N._I64x3(2048, 128, 60)), "16-byte"),
                     (dict(k_cache=pointers((1 << 20) + 8, 2 << 20)), "16-byte"), (dict(kc_stride=N._I64x3(2048, 0, 64)), "rows of a cache"),
                     (dict(v_cache=pointers((1 << 20) + 2048, 4 << 20)), "k_cache and v_cache"), (dict(k_cache=pointers(1 << 20, 3 << 20)), "layers")):
        err(compact(**kw), word)

    def release(**kw):
        a = N.ReleaseArgs()
        a.batch, a.page_size, a.table_pages, a.num_pages = 2, 16, 3, 4
        a.held_lens = a.kept_lens = a.block_table = a.pages = a.pages_released = 4096
        for k, v in kw.items():
            setattr(a, k, v)
        got = lib.fa_release_pages(ref(a), None), lib.fa_release_pages_checked(ref(a), ref(failed), None)
        assert got[0] == got[1]
        return got[0]
    for kw, word in ((dict(batch=-1), "negative"), (dict(page_size=0), "page_size"), (dict(pages=None), "pages"), (dict(held_lens=None), "held_lens"),
                     (dict(block_table=None), "block_table")):
        err(release(**kw), word)

    def norm(backward=False, **kw):
        a = N.QkNormArgs()
        a.batch, a.seqlen, a.heads_q, a.heads_kv, a.head_dim = 1, 2, 4, 2, 64
        for f in ("q", "k", "q_out", "k_out", "d_qo", "d_ko", "d_q", "d_k"):
            setattr(a, f, 4096)
        for f in ("q_stride", "k_stride", "qo_stride", "ko_stride", "d_qo_stride", "d_ko_stride", "d_q_stride", "d_k_stride"):
            setattr(a, f, N._I64x3(512, 256, 64))
        for k, v in kw.items():
            setattr(a, k, v)
        return (lib.fa_qk_norm_bwd if backward else lib.fa_qk_norm)(ref(a), None)
    for kw, word in ((dict(dtype=5), "dtype"), (dict(heads_q=0), "size"), (dict(head_dim=80), "head dimension"), (dict(cos=4096), "together"),
                     (dict(rotary_dim=66), "exceed"), (dict(rotary_dim=3), "exceed"), (dict(q=4096 + 8), "rows of q"),
                     (dict(k_stride=N._I64x3(512, 250, 64)), "rows of k"), (dict(q_out=None), "results"),
                     (dict(backward=True, d_ko=None), "gradients"), (dict(backward=True, d_q_weight=4096), "workspace")):
        err(norm(**kw), word)

    d = N.DecodeArgs()
    d.heads_q, d.heads_kv, d.head_dim, d.batch, d.seqlen_q, d.page_size, d.num_pages = 8, 2, 128, 1, 4, 64, 4
    d.q = d.o = d.k_cache = d.v_cache = d.cache_seqlens = d.tree_mask = 4096
    for f in ("q_stride", "o_stride", "kc_stride", "vc_stride"):
        setattr(d, f, N._I64x3(1024, 1024, 128))
    d.window_left, d.window_right = 100, -1
    err(lib.fa_decode_paged(ref(d), None), "tree_mask")
    d.window_left, d.alibi_slopes = -1, 4096
    err(lib.fa_decode_paged_checked(ref(d), ref(failed), None), "tree_mask")
    c = N.Cache8()
    c.code, c.block, c.k_scale, c.v_scale = 0, 16, 4096, 4096
    d.alibi_slopes = None
    err(lib.fa_decode_paged8(ref(d), ref(c), None), "16-bit")


def test_workspace_of_a_tree_grows_by_its_bits(native):
    N = native
    d = N.DecodeArgs()
    d.heads_q, d.heads_kv, d.head_dim, d.batch, d.seqlen_q, d.page_size, d.softmax_scale = 8, 2, 128, 300, 33, 64, 0.1
    assert N.lib().fa_decode_workspace_bytes(ctypes.byref(d)) == 0
    d.tree_mask = 4096
    assert N.lib().fa_decode_workspace_bytes(ctypes.byref(d)) >= 300 * 34 * 2 * 4
