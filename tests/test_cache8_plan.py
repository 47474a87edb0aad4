"""How calls on the 8-bit KV cache are cut, from the workspace that they ask for: no GPU."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def native():
    from flash_attn_triton_b200.build import build
    build()
    from flash_attn_triton_b200 import _native as N
    return N


# Bytes of the two rings of a CTA (stages x 16-bit tile + tiles of codes), where a merge keeps one float per piece and query row.
PAIR = {64: 6 * 16384 + 6 * 8192, 128: 3 * 32768 + 3 * 16384}                                # 256 rows
CHUNK = {64: 6 * 16384 + 8 * 8192, 128: 3 * 32768 + 5 * 16384, 256: 3 * 32768 + 3 * 16384}  # 128 rows


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_merges_have_room_for_their_pieces(native, dim):
    """The workspace of a chunk cut by keys is units * pieces * rows * (dim + 1) floats, and a few words."""
    N, lib = native, native.lib()
    seen = set()
    for heads_kv in (1, 2, 3):
        for group in (1, 2, 4, 7, 8, 16):
            for tokens in (17, 20, 32, 65, 129, 256, 700):
                for batch in (1, 2, 5):
                    for pages in (1, 40, 290, 600, 4000):
                        d, c = N.DecodeArgs(), N.Cache8()
                        d.batch, d.seqlen_q, d.heads_kv, d.heads_q, d.head_dim = batch, tokens, heads_kv, heads_kv * group, dim
                        d.page_size, d.num_pages, d.block_table_stride, d.block_table, d.softmax_scale = 256, 4 * pages, pages, 4096, 0.1
                        c.block = 256
                        pack = group if group & (group - 1) == 0 else 1
                        rows = tokens * pack
                        pair = dim <= 128 and rows > 128
                        per = 256 if pair else 128
                        units = batch * heads_kv * group // pack * -(-rows // per)
                        need = lib.fa_decode8_workspace_bytes(ctypes.byref(d), ctypes.byref(c))
                        pieces = need // (units * per * (dim + 1) * 4)
                        assert pieces * per * 4 <= (PAIR if pair else CHUNK)[dim], (heads_kv, group, tokens, batch, pages, pieces)
                        seen.add(pieces)
    assert 1 not in seen and {0, 4} <= seen and max(seen) > 100       # (0: not cut)
