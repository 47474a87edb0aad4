"""More of decoding with trees of drafted tokens; definitions and tolerances as in test_gpu_drafting.py."""
import math

import pytest
import torch

import drafting_reference as ref
import flash_attn_triton_b200 as fa
import test_gpu_drafting as base
from util import DEV

pytestmark = pytest.mark.gpu


# ---- nodes that only rows before them have in the mask -----------------------------------------------------------------------------
@base.WIDE
@pytest.mark.parametrize("spoil", [math.nan, math.inf])
@pytest.mark.parametrize("new", [False, True])
@pytest.mark.parametrize("splits", [0, 1])
@pytest.mark.parametrize("i", [1, 2, 3, 4, 5, 6, 7, 10, 11])
def test_nodes_that_causal_hides_may_hold_anything(i, splits, new, spoil, wide):
    """Masks with bits above the diagonal: rows of nodes that a request uses are all true, the others all false.  With `causal`, no row
    sees the nodes behind the last one in use."""
    dtype, lens, nodes, heads, heads_kv, dim, page, _ = case = base.TREES[i]
    gen = torch.Generator().manual_seed(500 + i)
    kc, vc, table, rows, where = base.make_cache(gen, dtype, lens, nodes, heads_kv, dim, page, capacity=base.wide_enough(case) if wide else 0)
    q, k, v = (base.rand(gen, len(lens), nodes, h, dim).to(dtype) for h in (heads, heads_kv, heads_kv))
    seen = torch.zeros(len(lens), nodes, nodes, dtype=torch.bool)
    for b in range(len(lens)):
        seen[b, :max(1, nodes // (2 + b))] = True
    sees = seen.tril()
    dead = ~sees.any(1)
    assert dead.any() and seen.any(1).all()
    k[dead], v[dead] = spoil, spoil
    kd, vd, lengths = kc.to(DEV), vc.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    if not new:
        for b, n in enumerate(lens):
            for p in range(nodes):
                kd[where(b, n + p)], vd[where(b, n + p)] = k[b, p].to(DEV), v[b, p].to(DEV)
    tokens = [k.to(DEV), v.to(DEV)] if new else []
    out = fa.flash_attn_with_kvcache(q.to(DEV), kd, vd, *tokens, cache_seqlens=lengths if new else lengths + nodes, causal=True, num_splits=splits,
                                     block_table=None if table is None else table.to(DEV), cache_batch_idx=None if rows is None else rows.to(DEV),
                                     tree_mask=seen.to(DEV))
    for b, n in enumerate(lens):
        place = [where(b, p) for p in range(n)]
        x, y = (torch.tensor([at[w] for at in place], dtype=torch.long) for w in range(2))
        every = torch.cat((torch.ones(nodes, n, dtype=torch.bool), sees[b]), 1)
        want, size = ref.attend(q[b], torch.cat((kc[x, y], k[b])), torch.cat((vc[x, y], v[b])), every, dim ** -0.5)
        base.within(out[b], want, base.half(dtype) * want.abs() + (base.half(dtype) + 2.0 ** -12) * size + 1e-6, ("out", b))
