"""More of decoding with trees of drafted tokens; definitions and tolerances as in test_gpu_drafting.py."""
import math
import os
import subprocess
import sys
import textwrap

import pytest
import torch

import drafting_reference as ref
import flash_attn_triton_b200 as fa
import test_gpu_drafting as base
from flash_attn_triton_b200 import drafting
from util import DEV

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


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


# ---- the first verification of a process -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("batch,nodes,vocab", [(160, 3, 6000), (64, 8, 24000), (30, 16, 47000)])
def test_first_verification_of_a_process(batch, nodes, vocab):
    """Shares of the vocabulary for which the kernel needs a little more than 48 KB of shared memory in all, its static part counted: nothing
    that an earlier call has asked for may be missing."""
    here = os.path.dirname(os.path.abspath(__file__))
    code = f"""
        import torch
        import test_gpu_drafting as base
        for dtype in (torch.float32, torch.float16, torch.bfloat16):
            given = base.verify_case(1, 2, {nodes}, {vocab}, dtype, 0.7)
            pick = torch.arange({batch}) % 2
            parents = given[1][pick]
            given = [x[pick] for x in given]
            base.check_verify([x[:2] for x in given], **{{"_%d" % i: (lambda y: lambda x: y.to(base.DEV))(y) for i, y in enumerate(given)}})
    """
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([here, os.path.dirname(here)]))
    done = subprocess.run([sys.executable, "-c", textwrap.dedent(code)], env=env, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


# ---- the step as it is written in drafting.py --------------------------------------------------------------------------------------
def test_the_documented_step_leaves_other_requests_alone():
    """Trees of different sizes in one call, and tables whose unused entries still name pages that other requests own (no call clears them):
    contexts stay as they were, accepted rows follow them, and every page has one owner."""
    gen = torch.Generator().manual_seed(9)
    batch, nodes, heads, heads_kv, dim, page, pool, vocab = 3, 40, 4, 2, 64, 16, 32, 61
    lens, nodes_of = [30, 16, 5], [nodes, 2, 1]
    order = torch.randperm(pool, generator=gen).to(torch.int32)
    table, at = torch.zeros(batch, 8, dtype=torch.int32), 0
    for b, n in enumerate(lens):
        held = -(-n // page)
        table[b, :held] = order[at:at + held]
        at += held
    for b in range(batch):                                    # behind each request's pages: those of the next one
        table[b, -(-lens[b] // page):] = table[(b + 1) % batch, 0]
    parents, seen = ref.tree(gen, batch, nodes, nodes_of)
    kc, vc = (base.rand(gen, pool, page, heads_kv, dim).to(F16) for _ in range(2))
    q, k, v = (base.rand(gen, batch, nodes, h, dim).to(F16) for h in (heads, heads_kv, heads_kv))
    draft = torch.softmax(base.rand(gen, batch, nodes, vocab), -1)
    angle = torch.outer(torch.arange(128.0), 100.0 ** (-torch.arange(0, dim, 2) / dim))
    at_gpu = dict(cache_seqlens=torch.tensor(lens, dtype=torch.int32), nodes_of=torch.tensor(nodes_of, dtype=torch.int32), free_pages=order[at:],
                  block_table=table, q=q, k=k, v=v, k_cache=kc, v_cache=vc, mask=seen, cos=angle.cos(), sin=angle.sin(),
                  depth=(seen.sum(-1) - 1).clamp_min(0).int(), draft_tokens=torch.randint(vocab, (batch, nodes), generator=gen), parents=parents,
                  target_probs=draft.clone(), draft_probs=draft, accept_uniforms=torch.zeros(batch, nodes),
                  sample_uniforms=torch.rand(batch, generator=gen))
    names = {n: x.clone().to(DEV) for n, x in at_gpu.items()}
    names.update(batch=batch, nodes=nodes, page_size=page, num_pages=pool, num_tokens=batch * nodes, q_weight=None, k_weight=None, torch=torch)
    names.update({n: getattr(fa, n) for n in ("build_block_table", "qk_norm_rotary", "flash_attn_with_kvcache", "verify_draft_tree",
                                              "kvcache_compact", "release_pages")})
    names["k_caches"], names["v_caches"] = [names["k_cache"]], [names["v_cache"]]
    step = [line for line in drafting.__doc__.splitlines() if line.startswith("    ")]
    assert len(step) == 7
    exec(textwrap.dedent("\n".join(step)), names)
    _, keys = fa.qk_norm_rotary(*(at_gpu[n].to(DEV) for n in ("q", "k")), None, None, names["cos"], names["sin"],
                                positions=torch.tensor(lens, device=DEV)[:, None] + names["depth"])
    keys, got_k, got_v, rows = keys.cpu(), names["k_cache"].cpu(), names["v_cache"].cpu(), names["block_table"].cpu()
    path, accepted = names["path"].cpu(), names["accepted"].tolist()
    assert max(accepted) > 2 and names["cache_seqlens"].tolist() == [n + m for n, m in zip(lens, accepted)]
    for b, n in enumerate(lens):
        for p in range(n):
            was, now = (int(table[b, p // page]), p % page), (int(rows[b, p // page]), p % page)
            assert torch.equal(got_k[now], kc[was]) and torch.equal(got_v[now], vc[was]), ("context", b, p)
        for i in range(accepted[b]):
            now = int(rows[b, (n + i) // page]), (n + i) % page
            assert torch.equal(got_k[now], keys[b, path[b, i]]) and torch.equal(got_v[now], v[b, path[b, i]]), ("accepted", b, i)
    owned = [x for b in range(batch) for x in rows[b, :-(-(lens[b] + accepted[b]) // page)].tolist()]
    free = names["free_pages"].tolist()[names["used"].item():] + names["pages"].tolist()[:names["n"].item()]
    assert sorted(owned + free) == list(range(pool))


# ---- gradients of gradients --------------------------------------------------------------------------------------------------------
def norm_call(leaf):
    return fa.qk_norm_rotary(leaf, leaf[..., :1, :])[0]


def refuses_second_gradients(call, leaf):
    """The first gradient is what it is without create_graph; a loss that reaches through it, whatever else is in it, is refused."""
    def first(**kw):
        return torch.autograd.grad(call(leaf).float().square().sum(), leaf, **kw)[0]
    want, got = first(), first(create_graph=True)
    assert torch.equal(got, want) and got.requires_grad and not want.requires_grad
    for loss in (got.float().square().sum(), got.float().sum() + leaf.float().square().sum()):
        with pytest.raises(RuntimeError, match="differentiated twice"):
            torch.autograd.grad(loss, leaf, retain_graph=True)
    # what does not reach through it has its gradient
    (g,) = torch.autograd.grad(got.detach().float().sum() + leaf.float().sum(), leaf)
    assert (g == 1).all()
    call(leaf).float().square().sum().backward(create_graph=True)
    assert torch.equal(leaf.grad, want)
    leaf.grad = None


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("behind", [0, 1])                     # 1: not on a 16-byte boundary, so that the call works on a copy
def test_gradients_of_gradients_of_the_norm_are_refused(dtype, behind):
    leaf = base.rand(torch.Generator().manual_seed(1), 2 * 5 * 3 * 64 + behind).to(dtype).to(DEV)[behind:].view(2, 5, 3, 64).requires_grad_()
    refuses_second_gradients(norm_call, leaf)


def test_gradients_of_gradients_of_the_norms_weights_are_refused():
    """dq depends on the weight also where q itself takes no gradient of its own, and the weight's gradient on the result's."""
    gen = torch.Generator().manual_seed(2)
    q, w, scale = base.rand(gen, 2, 5, 3, 64).to(DEV), torch.ones(64, device=DEV, requires_grad=True), torch.ones((), device=DEV, requires_grad=True)
    (g,) = torch.autograd.grad((fa.qk_norm_rotary(q, q, w, w)[0] * scale).sum(), w, create_graph=True)
    assert g.requires_grad
    with pytest.raises(RuntimeError, match="differentiated twice"):
        g.sum().backward()


def test_norm_under_function_transforms_is_refused():
    q = base.rand(torch.Generator().manual_seed(3), 4, 2, 5, 3, 64).to(DEV)
    with pytest.raises(RuntimeError):
        torch.vmap(lambda x: fa.qk_norm_rotary(x, x)[0])(q)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda x: fa.qk_norm_rotary(x, x)[0].sum())(q[0])
