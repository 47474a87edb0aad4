"""Windows far wider than any sequence (2^31 - 1 and above are usual words for "no bound") are as one that just covers it, bit for bit."""
import pytest
import torch

from test_gpu_cache8 import BF16, E4M3, F16, INT8, make_cache, make_table, rand
from util import DEV

pytestmark = pytest.mark.gpu

WIDE = [2 ** 30, 2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 62]


def fa():
    import flash_attn_triton_b200 as m
    return m


def windows(wide):
    return [((wide, wide), (5000, 5000)), ((wide, 0), (5000, 0)), ((7, wide), (7, 5000)), ((-1, wide), (-1, 5000))]


@pytest.mark.parametrize("wide", WIDE)
@pytest.mark.parametrize("lq,lk,dim", [(100, 100, 64), (300, 411, 128), (50, 20, 64), (70, 130, 256)])
def test_dense(lq, lk, dim, wide):
    q, k, v, do = (rand(i, 1, n, 2, dim).to(F16).to(DEV) for i, n in ((1, lq), (2, lk), (3, lk), (4, lq)))
    for got, same in windows(wide):
        outs = []
        for window in (got, same):
            x = [t.clone().requires_grad_() for t in (q, k, v)]
            out = fa().flash_attn_func_cross(*x, window_size=window) if lq != lk else fa().flash_attn_func(*x, window_size=window)
            outs.append([out, *torch.autograd.grad(out, x, do)])
        assert all(torch.equal(a, b) for a, b in zip(*outs)), got


@pytest.mark.parametrize("wide", WIDE)
def test_packed(wide):
    cu = torch.tensor([0, 70, 70, 300], dtype=torch.int32, device=DEV)
    q, k, v = (rand(i, 300, 2, 64).to(BF16).to(DEV) for i in range(3))
    for got, same in windows(wide):
        a, b = (fa().flash_attn_varlen_func(q, k, v, cu, cu, 230, 230, window_size=w) for w in (got, same))
        assert torch.equal(a, b), got


@pytest.mark.parametrize("wide", WIDE)
@pytest.mark.parametrize("code", [None, INT8, E4M3], ids=["16bit", "int8", "e4m3"])
@pytest.mark.parametrize("n,heads,dim", [(1, 4, 64), (5, 4, 128), (40, 4, 64), (100, 8, 128), (40, 4, 256)])
def test_cache(n, heads, dim, code, wide):
    """The second sequence is shorter than the chunk: rows in front of it."""
    page, lens = 16, [130, 3]
    table, pool = make_table(1, lens, page)
    kc, ks = make_cache(2, pool, page, 2, dim, code or INT8, 1)
    vc, vs = make_cache(3, pool, page, 2, dim, code or INT8, 1)
    kw = dict(k_scale=ks.to(DEV), v_scale=vs.to(DEV)) if code else {}
    if code is None:
        kc, vc = (x.float().mul(0.02).to(F16) for x in (kc, vc))
    q = rand(4, 2, n, heads, dim).to(F16).to(DEV)
    for got, same in windows(wide):
        a, b = (fa().flash_attn_with_kvcache(q, kc.to(DEV), vc.to(DEV), cache_seqlens=torch.tensor(lens, device=DEV), block_table=table.to(DEV),
                                             window_size=w, **kw) for w in (got, same))
        assert torch.equal(a, b), got
