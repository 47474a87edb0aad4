"""Decoding with trees of drafted tokens against its definition in 64 bits (drafting_reference.py): norms with the rotation, attention under a
tree's mask, verification, compaction and release of pages, and all of them in a row.

Tolerances.  `half(dtype)` is half a step of the output's type, relative to the value.  Norms: a mean of up to 256 squares is a chain of 13
roundings, its root and the reciprocal 3, the products and the rotation 4, each 2^-24 of what is added up: 2^-19 of that sum's size covers them
and the gradients' second mean.  Weight gradients: chains of up to 200 additions, 2^-16.  Attention: probabilities rounded to the type once, half a step
of sum p |v| beside that of the output; scores in fp32 (128 products of size 1 in units of the scale): 2^-12."""
import math
import threading

import pytest
import torch

import drafting_reference as ref
import flash_attn_triton_b200 as fa
from flash_attn_triton_b200 import _native as native
from util import DEV

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def half(dtype):
    return torch.finfo(dtype).eps / 2


def rand(gen, *shape):
    return torch.randn(*shape, generator=gen)


def within(got, want, bound, what):
    got = got.cpu().double()
    assert torch.isfinite(got).all(), what
    worst = ((got - want).abs() - bound).max().item() if want.numel() else 0.0
    assert worst <= 0.0, (what, worst, ((got - want).abs() / bound.clamp_min(1e-30)).max().item())


# ---- norms with the rotation -----------------------------------------------------------------------------------------------------
def norm_case(seed, dtype, lead, heads, heads_kv, dim, rotary, wide, longest=50):
    gen = torch.Generator().manual_seed(seed)
    q, k = (rand(gen, *lead, h, dim).mul(3).to(dtype) for h in (heads, heads_kv))
    w = F32 if wide else dtype
    qw, kw = ((1 + 0.3 * rand(gen, dim)).to(w) for _ in range(2))
    angle = torch.rand(longest, max(rotary // 2, 1), generator=gen, dtype=torch.float64) * 6.3
    cos, sin = (angle.cos().to(w), angle.sin().to(w)) if rotary else (None, None)
    return gen, q, k, qw, kw, cos, sin


def table_rows(table, positions, dim):
    """Rows of a table in doubles; positions outside it rotate nothing (cos 1, sin 0 come from the caller)."""
    inside = (positions >= 0) & (positions < table.shape[0])
    return table.double()[positions.clamp(0, table.shape[0] - 1)], inside[..., None]


NORMS = [
    # dtype, leading shape, heads, heads_kv, dim, rotary, interleaved, wide, positions
    (BF16, (2, 5), 4, 2, 128, 128, False, True, "batch"),
    (F16, (1, 1), 1, 1, 16, 16, False, False, None),
    (F16, (3, 7), 5, 1, 64, 32, False, True, "row"),
    (BF16, (1, 33), 32, 8, 128, 128, True, False, None),
    (F32, (2, 9), 3, 3, 256, 128, True, True, "batch"),
    (F32, (2, 19), 8, 2, 64, 64, False, True, None),
    (BF16, (13,), 7, 3, 32, 12, False, False, "packed"),      # halves of 6: pairs inside and across lanes
    (F16, (40,), 6, 2, 256, 200, True, True, "packed"),
    (F16, (2, 3), 9, 4, 16, 10, False, True, "one"),
    (BF16, (6, 3), 4, 4, 64, 0, False, False, None),          # no rotation
    (BF16, (0, 3), 4, 4, 64, 64, False, False, None),         # no tokens
    (BF16, (3, 0), 4, 4, 64, 64, False, False, None),
    (BF16, (2, 700), 10, 6, 128, 128, False, True, "batch"),  # several heads of a token per group of lanes
]


def run_norm(i, case, **change):
    dtype, lead, heads, heads_kv, dim, rotary, interleaved, wide, how = case
    gen, q, k, qw, kw, cos, sin = norm_case(i, dtype, lead, heads, heads_kv, dim, rotary, wide, longest=800)
    tokens = lead[-1]
    positions = None
    if how:
        shape = {"batch": lead, "row": (tokens,), "one": (1, tokens), "packed": lead}[how]
        positions = torch.randint(-3, 803, shape, generator=gen, dtype=torch.int64 if i % 2 else torch.int32)
    place = torch.arange(tokens).expand(lead) if positions is None else positions.long().expand(lead)
    gq, gk = rand(gen, *q.shape).to(dtype), rand(gen, *k.shape).to(dtype)
    leaves = [x.to(DEV).requires_grad_() for x in (q, k, qw, kw)]
    tables = [None if x is None else x.to(DEV) for x in (cos, sin)]
    out = fa.qk_norm_rotary(*leaves, *tables, positions=None if positions is None else positions.to(DEV), eps=1e-5,
                            rotary_interleaved=interleaved)
    grads = torch.autograd.grad(out, leaves, (gq.to(DEV), gk.to(DEV)))
    for x, g, weight, o, dx, dw in ((q, gq, qw, out[0], grads[0], grads[2]), (k, gk, kw, out[1], grads[1], grads[3])):
        assert o.dtype == dtype and dx.dtype == dtype and dw.dtype == weight.dtype and o.shape == x.shape and dx.shape == x.shape
        if rotary:
            (c, inside), (s, _) = table_rows(cos, place, dim), table_rows(sin, place, dim)
            c, s = torch.where(inside, c, 1.0), torch.where(inside, s, 0.0)
        else:
            c = s = torch.zeros(*lead, 0, dtype=torch.float64)
        want, size, wx, wx_size, ww, ww_size = ref.norm(x.double(), weight.double(), c, s, interleaved, float(torch.tensor(1e-5)), g.double())
        within(o, want, half(dtype) * want.abs() + 2.0 ** -19 * size + 1e-7, "out")
        within(dx, wx, half(dtype) * wx.abs() + 2.0 ** -18 * wx_size + 1e-7, "dx")
        within(dw, ww, half(weight.dtype) * ww.abs() + 2.0 ** -16 * ww_size + 1e-7, "dweight")
    return out, grads


@pytest.mark.parametrize("i", range(len(NORMS)))
def test_norm(i):
    run_norm(i, NORMS[i])


def test_norm_gradients_against_differences():
    """In fp32: a step of the loss along a direction is the gradient times that direction."""
    gen, q, k, qw, kw, cos, sin = norm_case(3, F32, (2, 6), 3, 2, 32, 24, True)
    gq, gk = rand(gen, *q.shape).to(DEV), rand(gen, *k.shape).to(DEV)
    leaves = [x.to(DEV).requires_grad_() for x in (q, k, qw, kw)]
    cos, sin = cos.to(DEV), sin.to(DEV)

    def loss(*x):
        a, b = fa.qk_norm_rotary(*x, cos, sin)
        return (a.double() * gq).sum() + (b.double() * gk).sum()
    grads = torch.autograd.grad(loss(*leaves), leaves)
    for i in range(4):
        d = rand(gen, *leaves[i].shape).to(DEV)
        h = 2.0 ** -7
        moved = [[x.detach() + (s * h * d if j == i else 0) for j, x in enumerate(leaves)] for s in (1, -1)]
        slope = (loss(*moved[0]) - loss(*moved[1])) / (2 * h)
        want = (grads[i].double() * d).sum()
        # third derivatives of size 1 times h^2, and fp32 noise of the outputs over h
        assert abs(slope - want) <= 2e-3 * (grads[i].double() * d).abs().sum() + 1e-3


def test_norm_is_the_same_every_time_and_over_strides():
    gen, q, k, qw, kw, cos, sin = norm_case(5, BF16, (2, 300), 8, 2, 128, 128, True, longest=300)
    packed = torch.cat((q, k, k), 2).to(DEV).requires_grad_()            # slices of a packed projection, read in place
    args = [qw.to(DEV).requires_grad_(), kw.to(DEV).requires_grad_(), cos.to(DEV), sin.to(DEV)]
    grads = []
    for x in (packed, packed, packed.detach().clone().requires_grad_()):
        a, b = fa.qk_norm_rotary(x[:, :, :8], x[:, :, 8:10], *args)
        grads.append((a, b, *torch.autograd.grad((a, b), (x, *args[:2]), (torch.ones_like(a), torch.ones_like(b)))))
    q2, k2 = q.to(DEV).requires_grad_(), k.to(DEV).requires_grad_()
    a, b = fa.qk_norm_rotary(q2, k2, *args)
    own = (a, b, *torch.autograd.grad((a, b), (q2, k2, *args[:2]), (torch.ones_like(a), torch.ones_like(b))))
    for g in grads[1:]:
        assert all(torch.equal(x, y) for x, y in zip(grads[0], g))
    assert torch.equal(own[0], grads[0][0]) and torch.equal(own[1], grads[0][1])
    assert torch.equal(own[2], grads[0][2][:, :, :8]) and torch.equal(own[3], grads[0][2][:, :, 8:10])
    assert (grads[0][2][:, :, 10:] == 0).all() and torch.equal(own[4], grads[0][3]) and torch.equal(own[5], grads[0][4])
    # gradients that are expanded, or come to one output alone; a row that is not 16-byte aligned; no weights
    y = fa.qk_norm_rotary(q2, k2, *args)
    g = torch.autograd.grad(y[0].sum(), (q2, k2), retain_graph=True)
    assert torch.equal(g[0], own[2]) and (g[1] == 0).all()
    odd = torch.zeros(2 * 300 * 8 * 128 + 1, dtype=BF16, device=DEV)[1:].view(2, 300, 8, 128)
    odd.copy_(q2.detach())
    assert torch.equal(fa.qk_norm_rotary(odd, k2, *args)[0], a)
    ones = torch.ones(128, dtype=BF16, device=DEV)
    assert torch.equal(fa.qk_norm_rotary(q2, k2)[0], fa.qk_norm_rotary(q2, k2, ones, ones)[0])


def test_norm_of_zeros_and_of_rows_that_are_no_numbers():
    """A row with an infinity has the norm of one: its numbers become 0, the infinity none."""
    q = torch.ones(1, 4, 2, 64, dtype=F16)
    q[0, 0] = 0
    q[0, 1, 0, 3], q[0, 2, 1, 7] = math.nan, math.inf
    x = q.to(DEV).requires_grad_()
    w = torch.ones(64, dtype=F16, device=DEV)
    a, b = fa.qk_norm_rotary(x, x, w, w)
    (g,) = torch.autograd.grad((a, b), (x,), (torch.ones_like(a), torch.ones_like(b)))
    assert (a[0, 0] == 0).all() and torch.isfinite(g[0, 0]).all()
    for out in (a, b):
        assert out[0, 1, 0].isnan().all() and torch.isfinite(out[0, 1, 1]).all() and torch.isfinite(out[0, 2, 0]).all() and (out[0, 3] == 1).all()
        assert out[0, 2, 1, 7].isnan() and (out[0, 2, 1, :7] == 0).all() and (out[0, 2, 1, 8:] == 0).all()
    angle = torch.zeros(4, 16, dtype=F16, device=DEV)
    out = fa.qk_norm_rotary(x, x, w, w, angle + 1, angle)[0]                                # the 32 that are not rotated, and the rest but the pair
    assert out[0, 2, 1, 7].isnan() and (out[0, 2, 1, 32:] == 0).all() and (out[0, 2, 1, 8:23] == 0).all()


# ---- attention under the mask of a tree -------------------------------------------------------------------------------------------
def make_cache(gen, dtype, lens, room, heads_kv, dim, page, pads=None, capacity=0):
    """Caches, paged from a shuffled pool or contiguous (page 0), and where position p of sequence b lies: (first index, row).  capacity: of a
    sequence, at least; with a large one a call takes the kernel for long caches."""
    if page == 0:
        rows = max(max(lens) + room + (max(pads) if pads else 0), capacity)
        kc, vc = (rand(gen, len(lens) + 1, rows, heads_kv, dim).to(dtype) for _ in range(2))
        order = torch.randperm(len(lens) + 1, generator=gen)[:len(lens)].to(torch.int32)
        return kc, vc, None, order, lambda b, p: (int(order[b]), p + (pads[b] if pads else 0))
    need = [-(-(n + room) // page) for n in lens]
    pool = torch.randperm(sum(need) + 2, generator=gen).to(torch.int32)
    table, at = torch.zeros(len(lens), max(max(need), -(-capacity // page)), dtype=torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = pool[at:at + n]
        table[b, n:] = pool[at]
        at += n
    kc, vc = (rand(gen, sum(need) + 2, page, heads_kv, dim).to(dtype) for _ in range(2))
    return kc, vc, table, None, lambda b, p: (int(table[b, p // page]), p % page)


TREES = [
    # dtype, lens, nodes, heads, heads_kv, dim, page, causal
    (F16, [0, 1, 130], 1, 8, 8, 128, 16, False),
    (BF16, [70, 0, 5], 4, 8, 4, 128, 16, False),
    (F16, [513, 64, 63], 7, 4, 2, 64, 48, False),
    (BF16, [300, 17], 33, 6, 3, 32, 16, False),
    (F16, [200, 90], 20, 4, 1, 16, 0, True),
    (BF16, [127, 128, 129, 0], 9, 8, 2, 128, 64, False),
    (F16, [1000, 3], 61, 8, 2, 64, 16, False),
    (BF16, [700, 120, 250], 33, 4, 1, 256, 32, True),
    (F16, [2500], 17, 8, 1, 128, 128, False),                 # pieces
    (BF16, [5000], 8, 4, 2, 256, 256, False),
    (F16, [90, 1300], 130, 2, 2, 128, 0, False),              # a tree over more than a tile of keys
    (BF16, [40, 260], 24, 14, 2, 64, 16, False),              # groups of 7
    (F16, [100, 31], 40, 8, 1, 128, 48, False),               # pages that a tile of keys does not consist of
]


def wide_enough(case):
    """A capacity with which a call of more than 8 query rows per head takes the kernel for long caches (more tiles than a few per SM)."""
    _, lens, nodes, heads, heads_kv, _, _, _ = case
    return 64 * 4 * 148 // (len(lens) * heads_kv * -(-nodes * heads // heads_kv // 16)) + 64


def run_tree(seed, case, new=True, used=None, spoil=None, mask=None, wide=False, pads=None, view=lambda x: x, **kw):
    dtype, lens, nodes, heads, heads_kv, dim, page, causal = case
    gen = torch.Generator().manual_seed(seed)
    kc, vc, table, rows, where = make_cache(gen, dtype, lens, nodes, heads_kv, dim, page, pads, wide_enough(case) if wide else 0)
    q, k, v = (rand(gen, len(lens), nodes, h, dim).to(dtype) for h in (heads, heads_kv, heads_kv))
    _, seen = ref.tree(gen, len(lens), nodes, used or [max(1, nodes - 3 * b) for b in range(len(lens))])
    if mask is not None:
        seen = mask(seen)
    if spoil is not None:                                     # what nobody sees may be no numbers
        dead = ~seen.any(1)
        k[dead], v[dead] = spoil, spoil
    scale = kw.pop("softmax_scale", dim ** -0.5)
    kd, vd = view(kc.to(DEV)), view(vc.to(DEV))
    if not new:
        for b, n in enumerate(lens):
            for i in range(nodes):
                kd[where(b, n + i)], vd[where(b, n + i)] = k[b, i].to(DEV), v[b, i].to(DEV)
    common = dict(block_table=None if table is None else table.to(DEV), cache_batch_idx=None if rows is None else rows.to(DEV),
                  softmax_scale=scale, causal=causal, tree_mask=seen.to(DEV),
                  cache_leftpad=torch.tensor(pads, dtype=torch.int32, device=DEV) if pads else None, **kw)
    if new:
        out = fa.flash_attn_with_kvcache(q.to(DEV), kd, vd, k.to(DEV), v.to(DEV), cache_seqlens=torch.tensor(lens, dtype=torch.int32, device=DEV), **common)
    else:
        out = fa.flash_attn_with_kvcache(q.to(DEV), kd, vd, cache_seqlens=torch.tensor(lens, dtype=torch.int32, device=DEV) + nodes, **common)
    got_k, got_v = kd.cpu(), vd.cpu()
    for b, n in enumerate(lens):
        place = [where(b, p) for p in range(n)]
        i, j = torch.tensor([x for x, _ in place], dtype=torch.long), torch.tensor([x for _, x in place], dtype=torch.long)
        sees = seen[b].tril() if causal else seen[b]
        sees = torch.cat((torch.ones(nodes, n, dtype=torch.bool), sees), 1)
        want, size = ref.attend(q[b], torch.cat((kc[i, j], k[b])), torch.cat((vc[i, j], v[b])), sees, scale)
        within(out[b], want, half(dtype) * want.abs() + (half(dtype) + 2.0 ** -12) * size + 1e-6, ("out", b))
        for p in range(nodes):                                # appended as they are
            for got, x, was in ((got_k, k, kc), (got_v, v, vc)):
                assert torch.equal(got[where(b, n + p)].view(torch.int16), x[b, p].view(torch.int16))
                was[where(b, n + p)] = got[where(b, n + p)]
    assert torch.equal(got_k.view(torch.int16), kc.view(torch.int16)) and torch.equal(got_v.view(torch.int16), vc.view(torch.int16))
    return out, seen


WIDE = pytest.mark.parametrize("wide", [False, True], ids=["few_tiles", "long_cache"])


@WIDE
@pytest.mark.parametrize("i", range(len(TREES)))
def test_tree(i, wide):
    run_tree(i, TREES[i], wide=wide)


@WIDE
@pytest.mark.parametrize("i", [1, 3, 6, 7, 10])
def test_tree_of_tokens_that_are_in_the_cache(i, wide):
    run_tree(100 + i, TREES[i], new=False, wide=wide)


@WIDE
@pytest.mark.parametrize("spoil", [math.nan, math.inf])
@pytest.mark.parametrize("new", [False, True])
@pytest.mark.parametrize("i", [1, 2, 3, 6, 7, 8, 9, 10, 12])
def test_nodes_that_nobody_sees_may_hold_anything(i, new, spoil, wide):
    lens, nodes = TREES[i][1], TREES[i][2]
    run_tree(200 + i, TREES[i], new=new, used=[max(1, nodes // 2)] + [1] * (len(lens) - 1), spoil=spoil, wide=wide)


@WIDE
@pytest.mark.parametrize("i", [1, 2, 3, 6, 7, 10])
def test_rows_that_see_nothing_and_any_mask(i, wide):
    """Without a context such rows are zeros; a mask need be no tree."""
    lens = [0] * len(TREES[i][1])
    case = (TREES[i][0], lens, *TREES[i][2:])
    gen = torch.Generator().manual_seed(i)
    _, seen = run_tree(300 + i, case, mask=lambda m: torch.rand(m.shape, generator=gen) < 0.3, wide=wide)
    out, seen = run_tree(310 + i, case, mask=lambda m: torch.zeros_like(m), wide=wide)
    assert (out == 0).all()


@WIDE
@pytest.mark.parametrize("i", [3, 4, 6, 10, 11])
def test_tree_in_caches_of_other_layouts(i, wide):
    """Contiguous ones with padding on the left, head-major ones, views of a larger tensor."""
    dtype, lens, nodes, heads, heads_kv, dim, page, causal = TREES[i]
    flat = (dtype, lens, nodes, heads, heads_kv, dim, 0, causal)
    for new in (True, False):
        run_tree(400 + i, flat, new=new, wide=wide, pads=[7 * b + 3 for b in range(len(lens))])
        run_tree(410 + i, TREES[i], new=new, wide=wide, view=lambda x: x.transpose(1, 2).contiguous().transpose(1, 2))
        run_tree(420 + i, TREES[i], new=new, wide=wide, view=lambda x: torch.cat((x, x, x), 2)[:, :, heads_kv:2 * heads_kv])


@WIDE
@pytest.mark.parametrize("kw", [dict(softmax_scale=-0.1), dict(softmax_scale=0.0), dict(num_splits=1), dict(num_splits=3)])
@pytest.mark.parametrize("i", [3, 6, 7])
def test_tree_with_other_scales_and_splits(i, kw, wide):
    run_tree(430 + i, TREES[i], wide=wide, **kw)


@pytest.mark.parametrize("dim,heads,nodes", [(64, 8, 16), (128, 8, 16), (256, 4, 12), (64, 8, 40), (128, 8, 40)])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_what_one_sequence_holds_reaches_no_other(dim, heads, nodes, value):
    """Contexts that are no numbers, in sequences that share a range with others: those come out bit for bit as without them."""
    gen = torch.Generator().manual_seed(dim + nodes)
    lens = [500, 130, 700, 90, 260, 40] * 6
    kc, vc, table, _, _ = make_cache(gen, BF16, lens, nodes, 2, dim, 16, capacity=6000)
    q, k, v = (rand(gen, len(lens), nodes, h, dim).to(BF16).to(DEV) for h in (heads, 2, 2))
    seen = ref.tree(gen, 1, nodes)[1][0].to(DEV)
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)

    def call(kc, vc):
        return fa.flash_attn_with_kvcache(q, kc.to(DEV), vc.to(DEV), k, v, cache_seqlens=lengths, block_table=table.to(DEV), tree_mask=seen)
    want = call(kc, vc)
    odd = [b for b in range(len(lens)) if b % 3 == 1]
    for what in range(2):
        cache = [kc.clone(), vc.clone()]
        for b in odd:
            cache[what][table[b, 1].item(), 3] = value
        got = call(*cache)
        rest = [b for b in range(len(lens)) if b not in odd]
        assert torch.equal(got[rest], want[rest]) and not torch.equal(got[odd], want[odd])


def test_tree_after_a_wait_that_ran_out():
    """The kernel for long caches is refused then, before anything is appended; the other one needs no waits."""
    dev = torch.cuda.current_device()
    assert native.lib().fa_debug_set_wait_status(dev, 31) == 0
    try:
        with pytest.raises(native.DeviceWaitError):
            run_tree(1, TREES[6], wide=True)
        run_tree(1, TREES[6], num_splits=1)
    finally:
        assert native.lib().fa_device_wait_clear(dev) == 0
    run_tree(1, TREES[6], wide=True)


@pytest.mark.parametrize("batch,longest,nodes,heads,heads_kv,dim,page", [
    (40, 700, 12, 4, 4, 64, 16),        # several sequences to a range, and the other way round
    (33, 300, 5, 8, 2, 128, 32),
    (200, 150, 20, 2, 2, 256, 64),      # more sequences than ranges
    (160, 400, 9, 2, 1, 128, 128),
    (300, 140, 40, 4, 1, 64, 0),        # two tiles of rows
    (3, 2000, 70, 32, 16, 64, 64),      # more units than SMs have room for at a time
    (2, 9000, 3, 8, 1, 128, 256),       # one unit, many ranges
])
def test_ranges_of_many_sequences(batch, longest, nodes, heads, heads_kv, dim, page):
    """How the sequences' tiles are cut into ranges: every place where a range may end.  Against the call for one sequence at a time, whose
    results are within the same bounds of the definition (test_tree)."""
    gen = torch.Generator().manual_seed(batch + nodes)
    lens = torch.randint(longest + 1, (batch,), generator=gen).tolist()
    lens[0], lens[-1] = 0, longest
    kc, vc, table, rows, _ = make_cache(gen, F16, lens, nodes, heads_kv, dim, page)
    kc, vc = kc.to(DEV), vc.to(DEV)
    q, k, v = (rand(gen, batch, nodes, h, dim).to(F16).to(DEV) for h in (heads, heads_kv, heads_kv))
    _, seen = ref.tree(gen, batch, nodes)
    seen, lengths = seen.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)

    def call(at):
        return fa.flash_attn_with_kvcache(q[at], kc, vc, k[at], v[at], cache_seqlens=lengths[at], tree_mask=seen[at],
                                          block_table=None if table is None else table.to(DEV)[at], cache_batch_idx=None if rows is None else rows.to(DEV)[at])
    out = call(slice(None))
    assert torch.equal(out, call(slice(None)))
    largest = v.abs().max().item() + vc.abs().max().item()
    for b in range(batch):
        want = call(slice(b, b + 1))[0].cpu().double()
        within(out[b], want, 2 * (half(F16) * want.abs() + (half(F16) + 2.0 ** -12) * largest), b)


def test_tree_masks_of_other_shapes():
    """One mask for all requests; rows of other strides.  A chain is the causal mask: bit for bit where the kernel is the same, few rows; else both
    results are within half a step of their own and (half + 2^-12) sum p |v| <= (half + 2^-12) max |v| of the same number (see the top), so
    within twice that of one another."""
    gen = torch.Generator().manual_seed(7)
    for nodes, heads, heads_kv, page in ((4, 8, 4, 16), (40, 8, 2, 64)):
        lens = torch.tensor([60, 200], dtype=torch.int32, device=DEV)
        kc, vc, table, _, _ = make_cache(gen, F16, [60, 200], nodes, heads_kv, 128, page, capacity=6000 if nodes > 4 else 0)
        q, k, v = (rand(gen, 2, nodes, h, 128).to(F16).to(DEV) for h in (heads, heads_kv, heads_kv))

        def call(**kw):
            return fa.flash_attn_with_kvcache(q, kc.to(DEV), vc.to(DEV), k, v, cache_seqlens=lens, block_table=table.to(DEV), **kw)
        seen = ref.tree(gen, 1, nodes)[1][0].to(DEV)
        want = call(tree_mask=seen.expand(2, -1, -1).contiguous())
        assert torch.equal(call(tree_mask=seen), want)
        assert torch.equal(call(tree_mask=seen.T.contiguous().T), want)
        wide = torch.zeros(2, nodes, nodes + 5, dtype=torch.bool, device=DEV)
        wide[:, :, 3:3 + nodes] = seen
        assert torch.equal(call(tree_mask=wide[:, :, 3:3 + nodes]), want)
        chain = torch.ones(nodes, nodes, dtype=torch.bool, device=DEV).tril()

        def same(got, want):
            if nodes == 4:
                assert torch.equal(got, want)
            else:
                largest = max(x.abs().max().item() for x in (vc.float(), v.float()))
                within(got, want.cpu().double(), 2 * half(F16) * (want.cpu().double().abs() + 2.0 ** -11) + 2 * (half(F16) + 2.0 ** -12) * largest, "chain")
        same(call(tree_mask=chain), call(causal=True))
        same(call(tree_mask=torch.ones_like(chain), causal=True), call(causal=True))
        same(call(tree_mask=torch.ones_like(chain)), call())
        assert torch.equal(call(tree_mask=torch.ones_like(chain), causal=True), call(tree_mask=chain))


def test_tree_refusals():
    q, c = torch.zeros(2, 4, 4, 64, dtype=F16, device=DEV), torch.zeros(2, 64, 2, 64, dtype=F16, device=DEV)
    lens, mask = torch.zeros(2, dtype=torch.int32, device=DEV) + 8, torch.ones(4, 4, dtype=torch.bool, device=DEV)
    for kw in (dict(tree_mask=mask.int()), dict(tree_mask=mask[:3]), dict(tree_mask=mask.cpu()), dict(tree_mask=mask.expand(3, 4, 4)),
               dict(tree_mask=mask, window_size=(5, 0)), dict(tree_mask=mask, alibi_slopes=torch.ones(4, device=DEV)),
               dict(tree_mask=mask, rotary_cos=torch.ones(64, 8, device=DEV, dtype=F16), rotary_sin=torch.ones(64, 8, device=DEV, dtype=F16))):
        with pytest.raises(ValueError):
            fa.flash_attn_with_kvcache(q, c, c, cache_seqlens=lens, **kw)
    codes, scale = torch.zeros(2, 64, 2, 64, dtype=torch.int8, device=DEV), torch.ones(2, 4, 2, device=DEV)
    with pytest.raises(ValueError, match="FP16 and BF16"):
        fa.flash_attn_with_kvcache(q, codes, codes.clone(), cache_seqlens=lens, k_scale=scale, v_scale=scale, tree_mask=mask)
    bad = torch.full((2, 4), 99, dtype=torch.int32, device=DEV)
    for nodes in (1, 4, 40):                                  # pages that do not exist, before anything is read
        x = torch.zeros(2, nodes, 4, 64, dtype=F16, device=DEV)
        with pytest.raises(ValueError, match="page"):
            fa.flash_attn_with_kvcache(x, c, c, cache_seqlens=lens, block_table=bad, tree_mask=torch.ones(nodes, nodes, dtype=torch.bool, device=DEV))


# ---- verification -----------------------------------------------------------------------------------------------------------------
def verify_case(seed, batch, nodes, vocab, dtype, near=1.0, sharp=2.0, branch=0.6, used=None):
    gen = torch.Generator().manual_seed(seed)
    parents, _ = ref.tree(gen, batch, nodes, used, branch)
    logits = sharp * rand(gen, batch, nodes, vocab).double()
    draft = torch.softmax(logits, -1)
    target = torch.softmax(logits + near * rand(gen, batch, nodes, vocab).double(), -1)
    tokens = torch.stack([torch.multinomial(draft[b, parents[b].clamp_min(0).long()], 1, generator=gen)[:, 0] for b in range(batch)])
    return [tokens, parents, target.to(dtype), draft.to(dtype), torch.rand(batch, nodes, generator=gen), torch.rand(batch, generator=gen)]


def check_verify(given, **views):
    dev = [x.to(DEV) for x in given]
    for i, view in views.items():
        dev[int(i[1:])] = view(dev[int(i[1:])])
    path, count, token = fa.verify_draft_tree(*dev)
    assert path.dtype == torch.int32 and count.dtype == torch.int32 and token.dtype == torch.int64
    tokens, parents, target, draft, accept, sample = given
    depths = []
    for b in range(target.shape[0]):
        want, after = ref.verify(tokens[b], parents if parents.ndim == 1 else parents[b], target[b], draft[b], accept[b], sample[b])
        assert path[b].tolist() == want + [-1] * (target.shape[1] - len(want)), b
        assert count[b].item() == len(want) and token[b].item() == after, (b, want, token[b].item(), after)
        depths.append(len(want))
    return depths


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("batch,nodes,vocab", [(1, 1, 1), (2, 1, 7), (3, 5, 33), (4, 9, 1000), (2, 40, 4097), (5, 16, 16391), (1, 7, 100003)])
def test_verify(batch, nodes, vocab, dtype):
    depths = []
    for seed, near, branch in ((1, 0.3, 0.6), (2, 1.5, 1.0), (3, 0.7, 0.0)):
        depths += check_verify(verify_case(seed, batch, nodes, vocab, dtype, near, branch=branch))
    assert nodes < 9 or vocab < 33 or max(depths) > 2


def test_verify_many_children_of_one_node():
    """Up to 63 rejections in a row, a long chain, a tree of 1024 nodes."""
    given = verify_case(5, 3, 64, 501, F32, near=3.0)
    given[1] = torch.tensor([-1] + [0] * 63, dtype=torch.int32)
    given[0] = torch.stack([torch.multinomial(given[3][b, 0].double(), 64, replacement=True) for b in range(3)])
    given[4] = 0.9 + 0.1 * given[4]
    check_verify(given)
    given = verify_case(6, 2, 1024, 65, F32, near=0.1, branch=0.02)
    check_verify(given)
    given[1] = torch.arange(-1, 1023, dtype=torch.int32)
    given[4] *= 0.05
    assert max(check_verify(given)) > 4


def test_verify_views_and_nodes_that_are_not_used():
    given = verify_case(8, 4, 12, 257, F32, used=[12, 7, 1, 3])
    check_verify(given)
    wide = lambda x: torch.nn.functional.pad(x, (0, 3))[..., :-3]                        # rows of another pitch
    check_verify(given, _2=wide, _3=lambda x: x.permute(2, 0, 1).contiguous().permute(1, 2, 0), _0=lambda x: x.int(), _1=lambda x: x.long())
    check_verify(given, _2=lambda x: x.transpose(0, 1).contiguous().transpose(0, 1), _4=lambda x: x.T.contiguous().T)
    given[1] = torch.where(given[1] >= 0, given[1], 2 ** 31 - 1)                          # no earlier node either
    check_verify(given)
    given[1] = torch.tensor([5, 0, 1, 3, -7, 2, 6, 1, 0, 11, 9, 3], dtype=torch.int32)    # nodes 3, 6, 9: before themselves or behind
    check_verify(given)
    given[0][:, 1], given[0][:, 2] = 257, -1                                              # tokens that do not exist are never accepted
    check_verify(given)


def test_verify_borders():
    """Numbers at the ends of [0, 1), distributions of one token or none, and such as are no numbers."""
    one = torch.zeros(1, 2, 8)
    p, q = one.clone(), one.clone()
    p[:, 0, 3], p[:, 1, 5], q[..., 2] = 1, 1, 1
    chain = torch.tensor([-1, 0], dtype=torch.int32)
    below = float(torch.nextafter(torch.tensor(1.0), torch.tensor(0.0)))
    for u in (0.0, below):
        for s in (0.0, below):
            args = [torch.tensor([[0, 2]]), chain, p, q, torch.full((1, 2), u), torch.full((1,), s)]
            assert check_verify(args) == [1]                  # the token has no mass in the target
            same = [torch.tensor([[0, 2]]), chain, q, q, torch.full((1, 2), u), torch.full((1,), s)]
            assert check_verify(same) == [2]                  # equal distributions: always accepted
    uneven = torch.rand(6, 3, 1009, generator=torch.Generator().manual_seed(1))
    uneven[:, :, :5], uneven[:, :, -5:] = 0, 0
    for s in (0.0, below, 0.5):
        args = [torch.zeros(6, 3, dtype=torch.int64), torch.tensor([-1, -1, -1], dtype=torch.int32), uneven, uneven, torch.rand(6, 3), torch.full((6,), s)]
        check_verify(args)
    # twice what is there: a rejection leaves nothing, and the target itself is what remains
    heavy = [torch.tensor([[0, 700]]), chain, uneven[:1, :2] * 0.25, uneven[:1, :2], torch.full((1, 2), 0.75), torch.full((1,), 0.3)]
    check_verify(heavy)
    for value in (0.0, math.nan, math.inf, -1.0):
        args = [torch.tensor([[0, 2]]), chain, torch.full((1, 2, 9), value), torch.full((1, 2, 9), 0.1), torch.full((1, 2), 0.5), torch.full((1,), 0.5)]
        path, count, token = fa.verify_draft_tree(*(x.to(DEV) for x in args))
        assert token.item() == -1 and path[0, 0].item() == 0
    none = [x[:0] for x in verify_case(1, 1, 3, 9, F32)]
    path, count, token = fa.verify_draft_tree(*(x.to(DEV) for x in none))
    assert path.shape == (0, 3) and count.shape == token.shape == (0,)


@pytest.mark.parametrize("batch,vocab", [(1, 300007), (160, 20011), (13, 40009), (16, 40009), (300, 9000)])
def test_verify_shares_that_shared_memory_has_no_room_for(batch, vocab):
    """A node is read again for every rejection, partly from shared memory; clusters of 1 to 8."""
    gen = torch.Generator().manual_seed(batch)
    base = torch.rand(4, 3, vocab, generator=gen)
    base[0] *= torch.rand(3, vocab, generator=gen) < 0.5      # zeros, as top-p leaves them
    base[1] *= 2.0 ** -140                                    # numbers below the smallest normal one
    p = base.clone()
    p[[0, 2]] /= base[[0, 2]].double().sum(-1, keepdim=True).float()
    q = torch.rand(3, vocab, generator=gen).double()
    q = (q / q.sum(-1, keepdim=True)).float()
    tokens, parents = torch.randint(vocab, (batch, 3), generator=gen), torch.tensor([-1, 0, 0], dtype=torch.int32)
    pick = torch.arange(batch) % 4
    check_verify([tokens, parents, p[pick], q.expand(batch, 3, vocab), 0.8 + 0.2 * torch.rand(batch, 3, generator=gen), torch.rand(batch, generator=gen)])
    # one number that is none, wherever it lies: no token follows
    spoilt = p[:2].clone()
    spoilt[0, 0, vocab - 1], spoilt[1, 0, 5] = math.nan, math.inf
    for up in (torch.full((3,), -1, dtype=torch.int32), parents):
        args = [torch.full((2, 3), 7), up, spoilt, q.expand(2, 3, vocab), torch.ones(2, 3), torch.rand(2, generator=gen)]
        args[2][:, 0, 7] = 0
        check_verify(args)
        assert (fa.verify_draft_tree(*(x.to(DEV) for x in args))[2] == -1).all()


def test_verify_from_two_threads():
    """Calls that need different amounts of shared memory, at the same time on streams of their own."""
    given = [[x.to(DEV) for x in verify_case(40 + i, batch, nodes, vocab, F32)] for i, (batch, nodes, vocab) in enumerate([(2, 6, 200003), (40, 3, 9001)])]
    want = [fa.verify_draft_tree(*x) for x in given]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(300):
                    got = fa.verify_draft_tree(*given[i])
                torch.cuda.current_stream().synchronize()
            assert all(torch.equal(x, y) for x, y in zip(got, want[i]))
        except BaseException as e:
            failed.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def test_verified_tokens_are_distributed_as_the_target():
    """20000 requests with the same distributions and independent numbers: the first token that comes out, accepted or sampled."""
    gen = torch.Generator().manual_seed(3)
    n, vocab = 20000, 6
    p, q = (torch.softmax(1.2 * rand(gen, vocab).double(), 0) for _ in range(2))
    parents = torch.tensor([-1, 0, 0, 0], dtype=torch.int32)
    tokens = torch.multinomial(q, 4 * n, replacement=True, generator=gen).view(n, 4)
    rows = lambda x: x.float().expand(n, 4, vocab).contiguous().to(DEV)
    path, count, token = fa.verify_draft_tree(tokens.to(DEV), parents.to(DEV), rows(p), rows(q), torch.rand(n, 4, generator=gen).to(DEV),
                                              torch.rand(n, generator=gen).to(DEV))
    first = torch.where(count.cpu() > 1, tokens.gather(1, path[:, 1:2].clamp_min(0).cpu().long())[:, 0], token.cpu())
    seen = torch.bincount(first, minlength=vocab).double() / n
    # five standard deviations of a share
    assert ((seen - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all(), (seen, p)
    assert (count > 1).float().mean() > (1 - (p - q).clamp_min(0).sum()) - 0.02


# ---- compaction -------------------------------------------------------------------------------------------------------------------
def compact_case(seed, dtype, lens, n, heads, dim, page, layers, accepted=None, pads=None):
    gen = torch.Generator().manual_seed(seed)
    _, _, table, rows, where = make_cache(gen, dtype, lens, n, 1, 16, page, pads)
    shape = (len(lens) + 1, max(lens) + n + (max(pads) if pads else 0)) if page == 0 else (int(sum(-(-(x + n) // page) for x in lens)) + 2, page)
    caches = [[rand(gen, *shape, heads, dim).to(dtype) for _ in range(layers)] for _ in range(2)]
    accepted = accepted or [int(torch.randint(n + 1, (1,), generator=gen)) for _ in lens]
    path = torch.full((len(lens), n), -9, dtype=torch.int32)
    for b, m in enumerate(accepted):
        path[b, :m] = torch.randperm(n, generator=gen)[:m].sort()[0]
    return caches, table, rows, where, path, accepted


def moved(caches, lens, path, accepted, where):
    out = [[c.clone() for c in one] for one in caches]
    for one in out:
        for c in one:
            for b, n in enumerate(lens):
                for i in range(accepted[b]):
                    c[where(b, n + i)] = c[where(b, n + int(path[b, i]))].clone()
    return out


@pytest.mark.parametrize("dtype,lens,n,heads,dim,page,layers", [
    (F16, [0], 1, 1, 16, 16, 1), (BF16, [5, 0, 31], 8, 4, 64, 16, 2), (F16, [15, 16, 17, 47], 33, 8, 128, 48, 3), (BF16, [100, 3], 70, 3, 256, 64, 2),
    (F16, [9, 2, 30], 12, 5, 32, 0, 2), (BF16, [40] * 30, 64, 2, 64, 32, 1), (F16, [7, 8], 150, 1, 128, 16, 2), (F16, [3], 5, 1, 16, 16, 131)])
@pytest.mark.parametrize("checks", [True, False])
def test_compact(dtype, lens, n, heads, dim, page, layers, checks):
    caches, table, rows, where, path, accepted = compact_case(n, dtype, lens, n, heads, dim, page, layers)
    want = moved(caches, lens, path, accepted, where)
    dev = [[c.to(DEV) for c in one] for one in caches]
    fa.set_validation(checks)
    try:
        fa.kvcache_compact(*dev, lens, path.to(DEV), torch.tensor(accepted, device=DEV), block_table=None if table is None else table.to(DEV),
                           cache_batch_idx=rows)
    finally:
        fa.set_validation(True)
    for got, one in zip(dev, want):
        assert all(torch.equal(g.cpu(), w) for g, w in zip(got, one))


def test_compact_views_and_left_padding():
    """Keys and values side by side in one tensor of all layers; rows behind padding."""
    pads, lens, n = [3, 0, 6], [4, 9, 0], 7
    caches, _, rows, where, path, accepted = compact_case(4, BF16, lens, n, 2, 64, 0, 2, accepted=[7, 4, 5], pads=pads)
    want = moved(caches, lens, path, accepted, where)
    pages, rows_of = caches[0][0].shape[:2]
    one = torch.zeros(pages, rows_of, 2, 2, 2, 64, dtype=BF16)                 # (page, row, layer, K or V, heads, dim)
    for w in range(2):
        for layer in range(2):
            one[:, :, layer, w] = caches[w][layer]
    dev = one.to(DEV)
    fa.kvcache_compact([dev[:, :, 0, 0], dev[:, :, 1, 0]], [dev[:, :, 0, 1], dev[:, :, 1, 1]], torch.tensor(lens, device=DEV), path.to(DEV).long(),
                       torch.tensor(accepted, device=DEV), cache_batch_idx=rows.to(DEV), cache_leftpad=torch.tensor(pads, device=DEV))
    for w in range(2):
        for layer in range(2):
            assert torch.equal(dev[:, :, layer, w].cpu(), want[w][layer])
    fa.kvcache_compact(dev[:, :, 0, 0], dev[:, :, 0, 1], [], path[:0].to(DEV), [])       # no requests


@pytest.mark.parametrize("batch", [3, 40])                     # checks in the kernel that moves, and in one ahead of it
@pytest.mark.parametrize("name,change,match", [
    ("accepted", lambda x: x.add_(100), "num_accepted"), ("accepted", lambda x: x.sub_(100), "num_accepted"),
    ("path", lambda x: x.copy_(x.flip(1)), "ascend"), ("path", lambda x: x[:, 3].copy_(x[:, 2]), "ascend"), ("path", lambda x: x[:, 0].fill_(-1), "ascend"),
    ("path", lambda x: x[:, -1].fill_(2 ** 31 - 1), "inside"), ("lens", lambda x: x.sub_(1000), "inside"), ("lens", lambda x: x.add_(2 ** 30), "inside"),
    ("table", lambda x: x.add_(1000), "exist"), ("table", lambda x: x.sub_(1000), "exist")])
def test_compact_refusals_by_value(batch, name, change, match):
    """One request of all is wrong: nothing is moved; without checks, only that request is passed over."""
    lens, n = [20 + b for b in range(batch)], 16
    caches, table, _, where, path, _ = compact_case(1, F16, lens, n, 2, 64, 16, 1, accepted=[n - 2] * batch)
    path[:, n - 2:] = path[:, n - 3:n - 2] + torch.arange(1, 3)
    accepted = [n - 2] * batch
    if name == "path" and match == "inside":
        accepted = [n] * batch
        path[:] = torch.arange(n)
    which = batch // 2
    given = dict(lens=torch.tensor(lens, dtype=torch.int32), table=table, path=path.clone(), accepted=torch.tensor(accepted, dtype=torch.int32))
    change(given[name][which:which + 1] if given[name].ndim == 2 else given[name][which:which + 1])
    given = {k: v.to(DEV) for k, v in given.items()}
    dev = [[c.to(DEV) for c in one] for one in caches]

    def call():
        fa.kvcache_compact(*dev, given["lens"], given["path"], given["accepted"], block_table=given["table"])
    with pytest.raises(ValueError, match=match):
        call()
    assert all(torch.equal(g.cpu(), c) for got, one in zip(dev, caches) for g, c in zip(got, one))
    fa.set_validation(False)
    try:
        call()
    finally:
        fa.set_validation(True)
    accepted[which] = 0
    want = moved(caches, lens, path, accepted, where)
    assert all(torch.equal(g.cpu(), c) for got, one in zip(dev, want) for g, c in zip(got, one))


def test_compact_refuses_caches_that_overlap():
    c = torch.zeros(4, 16, 2, 64, dtype=F16, device=DEV)
    path, one = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    for k, v in ((c, c), ([c, c], [c.clone(), c.clone()]), (c[:2], c[1:3]), (c[:, :1].expand(4, 16, 2, 64), c.clone())):
        with pytest.raises(ValueError, match="overlap"):
            fa.kvcache_compact(k, v, one, path, one)


# ---- pages ------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("batch,page,longest,extra", [(1, 16, 5, 0), (7, 16, 100, 3), (300, 24, 500, 0), (2100, 1, 9, 50), (5, 256, 9000, 1)])
def test_release(batch, page, longest, extra):
    gen = torch.Generator().manual_seed(batch)
    held = torch.randint(longest + 1, (batch,), generator=gen)
    kept = (held * torch.rand(batch, generator=gen)).long() * (torch.rand(batch, generator=gen) < 0.7)
    kept = torch.where(torch.rand(batch, generator=gen) < 0.2, held, kept)
    width = -(-longest // page) + 2
    table = torch.randint(10 ** 6, (batch, width + 3), generator=gen, dtype=torch.int32)[:, :width]
    want = [p for b in range(batch) for p in table[b, -(-int(kept[b]) // page):-(-int(held[b]) // page)].tolist()]
    dev = table.to(DEV)
    pages, n = fa.release_pages(held.to(DEV), kept.int().to(DEV), dev, page, len(want) + extra)
    assert pages.tolist() == want + [-1] * extra and n.item() == len(want) and pages.dtype == n.dtype == torch.int32
    assert torch.equal(dev.cpu(), table)


def test_release_refusals_by_value():
    table = torch.arange(12, dtype=torch.int32, device=DEV).view(3, 4)
    for held, kept, room, match in (([9, 9, 9], [1, -1, 1], 9, "negative"), ([9, 9, 9], [1, 10, 1], 9, "larger"), ([9, 65, 9], [1, 1, 1], 9, "row"),
                                    ([64, 64, 64], [0, 0, 0], 11, "num_pages")):
        with pytest.raises(ValueError, match=match):
            fa.release_pages(held, kept, table, 16, room)
        fa.set_validation(False)
        try:
            pages, n = fa.release_pages(held, kept, table, 16, room)
        finally:
            fa.set_validation(True)
        assert (pages == -1).all() and n.item() == -1
    pages, n = fa.release_pages([], [], table[:0], 16, 2)
    assert pages.tolist() == [-1, -1] and n.item() == 0
    assert fa.release_pages([16, 0, 1], [16, 0, 1], table, 16, 0)[1].item() == 0


# ---- together ---------------------------------------------------------------------------------------------------------------------
def test_steps_of_drafting_and_verifying():
    """Three steps of five requests through build_block_table, norms, appends, attention, verification, compaction and release, against the
    same from plain lists of keys: the caches then hold what a run without drafts would have put there, and no page is lost."""
    gen = torch.Generator().manual_seed(11)
    B, N, H, HK, D, page, vocab, layers, pool = 5, 12, 4, 2, 64, 16, 97, 2, 64
    lens = torch.tensor([30, 0, 15, 16, 47], dtype=torch.int32)
    free = torch.randperm(pool, generator=gen).to(torch.int32)
    table = torch.zeros(B, 8, dtype=torch.int32, device=DEV)
    caches = [[torch.zeros(pool, page, HK, D, dtype=BF16, device=DEV) for _ in range(layers)] for _ in range(2)]
    weight = (1 + 0.2 * rand(gen, D)).to(BF16).to(DEV)
    angle = torch.outer(torch.arange(200.0), 100.0 ** (-torch.arange(0, D, 2) / D))
    cos, sin = angle.cos().to(DEV), angle.sin().to(DEV)
    held = [[[] for _ in range(B)] for _ in range(layers)]    # (key, value) of every token of a request
    slots, _, used = fa.build_block_table(torch.zeros(B), lens, free, table, page, int(lens.sum()))
    free = free[used.item():]
    seq = torch.repeat_interleave(torch.arange(B), lens.long())
    for layer in range(layers):
        x = rand(gen, len(seq), 2, HK, D).to(BF16)
        for w in range(2):
            caches[w][layer].view(-1, HK, D)[slots] = x[:, w].to(DEV)
        for i, b in enumerate(seq.tolist()):
            held[layer][b].append((x[i, 0], x[i, 1]))
    for step in range(3):
        parents, seen = ref.tree(gen, B, N, [N, N - 3, N, 1, N - 5])
        depth = (seen.sum(-1) - 1).clamp_min(0)
        dev_lens = lens.to(DEV)
        _, _, used = fa.build_block_table(dev_lens, torch.full((B,), N), free, table, page, B * N)
        taken, free = free[:used.item()], free[used.item():]
        tree_kv = []
        for layer in range(layers):
            q, k, v = (rand(gen, B, N, h, D).to(BF16).to(DEV) for h in (H, HK, HK))
            qr, kr = fa.qk_norm_rotary(q, k, weight, weight, cos, sin, positions=dev_lens[:, None] + depth.to(DEV))
            c, s = (x.cpu().double()[lens[:, None].long() + depth] for x in (cos, sin))
            want, size = ref.norm(k.cpu().double(), weight.cpu().double(), c, s, False, 1e-6)
            within(kr, want, half(BF16) * want.abs() + 2.0 ** -19 * size + 1e-7, "rotated keys")
            out = fa.flash_attn_with_kvcache(qr, caches[0][layer], caches[1][layer], kr, v, cache_seqlens=dev_lens, block_table=table,
                                             tree_mask=seen.to(DEV))
            kr, v, qr = kr.cpu(), v.cpu(), qr.cpu()
            for b in range(B):
                keys = torch.stack([x for x, _ in held[layer][b]] + list(kr[b]))
                vals = torch.stack([x for _, x in held[layer][b]] + list(v[b]))
                sees = torch.cat((torch.ones(N, int(lens[b]), dtype=torch.bool), seen[b]), 1)
                want, size = ref.attend(qr[b], keys, vals, sees, D ** -0.5)
                within(out[b], want, half(BF16) * want.abs() + (half(BF16) + 2.0 ** -12) * size + 1e-6, "attention")
            tree_kv.append((kr, v))
        given = verify_case(20 + step, B, N, vocab, F32, near=0.4)
        given[1] = parents
        given[0] = torch.stack([torch.multinomial(given[3][b, parents[b].clamp_min(0).long()].double(), 1, generator=gen)[:, 0] for b in range(B)])
        check_verify(given)
        path, accepted, token = fa.verify_draft_tree(*(x.to(DEV) for x in given))
        fa.kvcache_compact(*caches, dev_lens, path, accepted, block_table=table)
        back, n = fa.release_pages(dev_lens + N, dev_lens + accepted, table, page, len(taken))
        free = torch.cat((free, back[:n.item()].cpu()))
        for b in range(B):
            for layer in range(layers):
                held[layer][b] += [(tree_kv[layer][0][b, i], tree_kv[layer][1][b, i]) for i in path[b, :accepted[b]].tolist()]
        lens = lens + accepted.cpu()
        rows = table.cpu()
        for b in range(B):
            assert len(held[0][b]) == lens[b]
            for layer in range(layers):
                for p, (key, value) in enumerate(held[layer][b]):
                    at = int(rows[b, p // page]), p % page
                    assert torch.equal(caches[0][layer][at].cpu(), key) and torch.equal(caches[1][layer][at].cpu(), value)
        owned = [p for b in range(B) for p in rows[b, :-(-int(lens[b]) // page)].tolist()]
        assert sorted(owned + free.tolist()) == list(range(pool))


def test_streams_and_graphs():
    """All calls captured into a graph on a stream of its own and replayed beside the same calls on another stream."""
    gen = torch.Generator().manual_seed(2)
    B, N = 3, 20
    kc, vc, table, _, _ = make_cache(gen, F16, [500, 40, 3000], N, 2, 128, 64, capacity=5000)
    lens = torch.tensor([500, 40, 3000], dtype=torch.int32, device=DEV)
    q, k, v = (rand(gen, B, N, h, 128).to(F16).to(DEV) for h in (8, 2, 2))
    _, seen = ref.tree(gen, B, N)
    table, seen = table.to(DEV), seen.to(DEV)
    angle = torch.rand(4000, 64, generator=gen).to(DEV)
    given = [x.to(DEV) for x in verify_case(4, B, N, 5000, F32)]
    positions = lens[:, None] + torch.arange(N, device=DEV, dtype=torch.int32)

    def step(cache, leaf):
        qr, kr = fa.qk_norm_rotary(leaf, k, None, None, angle, angle, positions=positions)
        out = fa.flash_attn_with_kvcache(qr.detach(), *cache, kr.detach(), v, cache_seqlens=lens, block_table=table, tree_mask=seen)
        path, n, token = fa.verify_draft_tree(*given)
        fa.kvcache_compact(*cache, lens, path, n, block_table=table)
        pages = fa.release_pages(lens + N, lens + n, table, 64, 8)
        return (out, path, n, token, *pages, *torch.autograd.grad(qr, leaf, out))
    fa.set_validation(False)
    try:
        want_cache = [kc.to(DEV), vc.to(DEV)]
        want = step(want_cache, q.clone().requires_grad_())
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        caches = [[kc.to(DEV), vc.to(DEV)] for _ in range(2)]
        leaves = [q.clone().requires_grad_() for _ in range(2)]
        torch.cuda.synchronize()
        graphs, outs = [], []
        for s, c, leaf in zip(streams, caches, leaves):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                outs.append(step(c, leaf))
            graphs.append(graph)
        for _ in range(3):
            for c in caches:
                c[0].copy_(kc.to(DEV))
                c[1].copy_(vc.to(DEV))
            torch.cuda.synchronize()
            for s, graph in zip(streams, graphs):
                with torch.cuda.stream(s):
                    graph.replay()
            torch.cuda.synchronize()
            for c, out in zip(caches, outs):
                assert all(torch.equal(x, y) for x, y in zip(out, want)) and all(torch.equal(x, y) for x, y in zip(c, want_cache))
    finally:
        fa.set_validation(True)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):             # checks need the host
        for call in (lambda: fa.kvcache_compact(*want_cache, lens, want[1], want[2], block_table=table),
                     lambda: fa.release_pages(lens + N, lens, table, 64, 8)):
            with pytest.raises(RuntimeError, match="captured"):
                call()
