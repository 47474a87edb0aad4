"""KV cache in 8 bits: append, attention, block tables, and a serving loop of the three."""
import math

import numpy as np
import pytest
import torch

import cache8_reference as ref
from util import DEV

pytestmark = pytest.mark.gpu

INT8, E4M3 = torch.int8, torch.float8_e4m3fn
F16, BF16 = torch.float16, torch.bfloat16


def fa():
    import flash_attn_triton_b200 as m
    return m


def rand(seed, *shape):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal(shape, dtype=np.float32))


def make_cache(seed, pages, page, heads, dim, code, blocks):
    x = rand(seed, pages, page, heads, dim) * (ref.LARGEST[code] / 3.5)
    scale = torch.from_numpy(np.random.default_rng(seed + 1).uniform(0.3, 1.6, (pages, blocks, heads)).astype(np.float32))
    return ref.coded(x, code), scale * (3.5 / ref.LARGEST[code])


def make_table(seed, lens, page, spare=1):
    """Block table over a shuffled pool, and the pool's size; rows end in copies of their first page."""
    need = [-(-n // page) for n in lens]
    order = np.random.default_rng(seed).permutation(sum(need) + spare).astype(np.int32)
    table = np.zeros((len(lens), max(1, max(need))), dtype=np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b] = order[min(at, len(order) - 1)]
        table[b, :n] = order[at:at + n]
        at += n
    return torch.from_numpy(table), sum(need) + spare


def slots_of(table, old, new, page):
    out = []
    for b, (n, m) in enumerate(zip(old, new)):
        out += [int(table[b, p // page]) * page + p % page for p in range(n, n + m)]
    return torch.tensor(out, dtype=torch.int64)


def same_cache(got, want):
    assert torch.equal(ref.bits(got.cpu()), ref.bits(want))


# ---- append --------------------------------------------------------------------------------------------------------
APPENDS = [
    # old lengths, new tokens, page, blocks, heads, dim
    ([0, 0, 0], [1, 1, 1], 16, 1, 1, 64),
    ([5, 16, 31, 0], [1, 1, 1, 1], 16, 1, 4, 128),
    ([0, 3, 17], [40, 1, 77], 24, 3, 2, 32),
    ([7, 250, 0], [300, 13, 1], 256, 1, 3, 128),
    ([1, 100], [500, 130], 128, 2, 2, 256),
    ([0, 9, 2], [33, 0, 5], 8, 8, 5, 16),             # a scale per token
    ([3], [1000], 1024, 1, 1, 64),                    # the largest block
    ([0] * 40, [1 + 13 * (i % 5) for i in range(40)], 32, 2, 8, 64),
]


@pytest.mark.parametrize("code", [INT8, E4M3], ids=["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(case, dtype, code):
    old, new, page, blocks, heads, dim = APPENDS[case]
    table, pool = make_table(case, [n + m for n, m in zip(old, new)], page)
    slots = slots_of(table, old, new, page)
    k, v = rand(100 + case, len(slots), heads, dim).to(dtype), (3 * rand(200 + case, len(slots), heads, dim)).to(dtype)
    kc, ks = make_cache(300 + case, pool, page, heads, dim, code, blocks)
    vc, vs = make_cache(400 + case, pool, page, heads, dim, code, blocks)
    got = [t.to(DEV) for t in (kc, vc, ks, vs)]
    fa().kvcache_append(k.to(DEV), v.to(DEV), got[0], got[1], slots.to(DEV), got[2], got[3])
    ref.append_slots(k, kc, ks, slots)
    ref.append_slots(v, vc, vs, slots)
    same_cache(got[0], kc)
    same_cache(got[1], vc)
    assert torch.equal(got[2].cpu(), ks) and torch.equal(got[3].cpu(), vs)
    # and a value that has just been written is within half a step of its code
    size = page // blocks
    for cache, scale, x in ((kc, ks, k), (vc, vs, v)):
        held = ref.values(cache, scale).flatten(0, 1)[slots]
        step = scale.repeat_interleave(size, dim=1).flatten(0, 1)[slots].double()[..., None]
        half = step / 2 if code == INT8 else torch.maximum(x.double().abs() * 2.0 ** -4, step * 2.0 ** -10)
        last = torch.ones(len(slots), dtype=torch.bool)
        assert ((held - x.double()).abs() <= half * (1 + 1e-5))[last].all()


def test_append_strided_and_padded():
    """Slices of a packed projection, caches inside larger tensors, slots of -1 between and behind the tokens."""
    page, heads, dim, pool = 16, 3, 64, 9
    big = rand(1, 50, 3, heads, dim).to(BF16).to(DEV)
    k, v = big[:, 1], big[:, 2]
    both = torch.randint(-127, 128, (pool, page, 2, heads, dim), dtype=torch.int8, device=DEV)
    kc, vc = both[:, :, 0], both[:, :, 1]
    scales = torch.rand(2, heads, pool, 2, device=DEV)
    ks, vs = scales[0].permute(1, 2, 0), scales[1].permute(1, 2, 0)
    slots = torch.cat([torch.arange(20, 41), torch.tensor([-1, -7]), torch.arange(64, 80), torch.tensor([3 * 16 + 7] + [-1] * 10)])
    assert len(slots) == 50
    want = [t.cpu().contiguous() for t in (kc, vc, ks, vs)]
    fa().kvcache_append(k, v, kc, vc, slots.to(torch.int32).to(DEV), ks, vs)
    ref.append_slots(k.cpu(), want[0], want[2], slots)
    ref.append_slots(v.cpu(), want[1], want[3], slots)
    for got, w in zip((kc, vc, ks, vs), want):
        assert torch.equal(got.cpu(), w)


@pytest.mark.parametrize("code", [INT8, E4M3], ids=["int8", "e4m3"])
def test_append_of_zeros_infinities_and_nan(code):
    """Zeros have scale 0; an infinity or NaN spoils the values of its block and head, and nothing else; a fresh start heals it."""
    page, heads, dim = 16, 2, 32
    kc, ks = make_cache(5, 6, page, heads, dim, code, 1)
    x = rand(6, 4 * page, heads, dim).to(F16)
    x[:page] = 0
    x[page + 3, 1, 7] = math.inf
    x[2 * page + 5, 0, 9] = math.nan
    x[3 * page:, 0] = 6e-8                            # smallest numbers of fp16
    kd, vd, ksd, vsd = kc.to(DEV), kc.to(DEV), ks.to(DEV), ks.to(DEV)
    slots = torch.arange(page, 5 * page)
    fa().kvcache_append(x.to(DEV), x.to(DEV), kd, vd, slots.to(DEV), ksd, vsd)
    s = ksd.cpu()
    assert (s[1] == 0).all() and math.isinf(s[2, 0, 1]) and math.isnan(s[3, 0, 0])
    held = ref.values(kd.cpu(), s)
    assert (held[1] == 0).all()
    assert not torch.isfinite(held[2, :, 1]).any() and not torch.isfinite(held[3, :, 0]).any()
    want, wants = kc.clone(), ks.clone()
    ref.append_slots(x, want, wants, slots)
    for page_, head in ((1, 0), (1, 1), (2, 0), (3, 1), (4, 0), (4, 1), (0, 0), (5, 1)):
        assert torch.equal(ref.bits(kd.cpu()[page_, :, head]), ref.bits(want[page_, :, head])) and s[page_, 0, head] == wants[page_, 0, head]
    fine = rand(7, page, heads, dim).to(F16)
    fa().kvcache_append(fine.to(DEV), fine.to(DEV), kd, vd, torch.arange(3 * page, 4 * page, device=DEV), ksd, vsd)
    assert torch.isfinite(ref.values(kd.cpu(), ksd.cpu())[3]).all()


def test_append_raises_scales_step_by_step():
    """One token at a time into one block, each larger than all before: every value stays within the steps of its roundings."""
    page, heads, dim, n = 32, 2, 64, 32
    for code in (INT8, E4M3):
        kc, ks = make_cache(8, 2, page, heads, dim, code, 1)
        kd, vd, ksd, vsd = kc.to(DEV), kc.to(DEV), ks.to(DEV), ks.to(DEV)
        x = (rand(9, n, heads, dim).clamp(-3, 3) * torch.linspace(0.5, 4, n)[:, None, None]).to(F16)
        for i in range(n):
            fa().kvcache_append(x[i:i + 1].to(DEV), x[i:i + 1].to(DEV), kd, vd, torch.tensor([page + i], device=DEV), ksd, vsd)
            ref.append_run(x[i:i + 1], kc, ks, 1, i)
        same_cache(kd, kc)
        assert torch.equal(ksd.cpu(), ks)


# ---- attention -------------------------------------------------------------------------------------------------------
def run_attend(seed, old, n, append, heads, heads_kv, dim, page, blocks, dtype, code, paged=True, rows=None, leftpad=None, q_gain=1.0, **kw):
    """One call against the reference; returns the largest error over its tolerance."""
    B = len(old)
    new = n if append is True else int(append or 0)
    lens = [x + new for x in old]
    place = {}
    if paged:
        table, pool = make_table(seed, [max(1, x) for x in lens], page)
        place["table"] = table
    else:
        pool = B if rows is None else max(rows) + 2
        if rows is not None:
            place["batch_idx"] = torch.tensor(rows)
        if leftpad is not None:
            place["leftpad"] = torch.tensor(leftpad)
    kc, ks = make_cache(seed + 10, pool, page, heads_kv, dim, code, blocks)
    vc, vs = make_cache(seed + 20, pool, page, heads_kv, dim, code, blocks)
    q = (q_gain * rand(seed + 30, B, n, heads, dim)).to(dtype)
    k = v = None
    if new:
        k, v = rand(seed + 40, B, new, heads_kv, dim).to(dtype), (2 * rand(seed + 50, B, new, heads_kv, dim)).to(dtype)
    d = lambda t: None if t is None else t.to(DEV)
    kd, vd, ksd, vsd = d(kc), d(vc), d(ks), d(vs)
    out = fa().flash_attn_with_kvcache(
        d(q), kd, vd, d(k), d(v), cache_seqlens=torch.tensor(old, dtype=torch.int32, device=DEV), block_table=d(place.get("table")),
        cache_batch_idx=d(place.get("batch_idx")), cache_leftpad=d(place.get("leftpad")), k_scale=ksd, v_scale=vsd, **kw)
    if new:
        ref.append_call(k, kc, ks, old, **place)
        ref.append_call(v, vc, vs, old, **place)
        same_cache(kd, kc)
        same_cache(vd, vc)
        assert torch.equal(ksd.cpu(), ks) and torch.equal(vsd.cpu(), vs)
    kv, vv = ref.values(kc, ks), ref.values(vc, vs)
    alibi = kw.get("alibi_slopes")
    if alibi is not None:
        alibi = torch.as_tensor(alibi).cpu().expand(B, heads)
    want, weight = ref.attend(q, kv, vv, lens, kw.get("softmax_scale"), kw.get("causal", False), kw.get("window_size", (-1, -1)), alibi, **place)
    assert out.dtype == dtype and out.shape == q.shape
    got = out.double().cpu()
    assert torch.isfinite(got).all()
    tol = ref.tolerance(want, weight, dtype, max(lens), float(vv.abs().max()))
    ratio = ((got - want).abs() / tol).max().item()
    assert ratio <= 1.0, ratio
    return ratio


@pytest.mark.parametrize("code", [INT8, E4M3], ids=["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("dim", [16, 32, 64, 128, 256])
def test_attend_dims(dim, dtype, code):
    run_attend(dim, [0, 1, 63, 64, 200], 1, True, 8, 2, dim, 16, 2, dtype, code, causal=True)
    run_attend(dim + 1, [130, 7], 3, True, 4, 1, dim, 32, 2, dtype, code, causal=True)


ATTENDS = [
    dict(old=[1], n=1, append=0, heads=1, heads_kv=1, dim=64, page=16, blocks=1),
    dict(old=[2000], n=1, append=True, heads=32, heads_kv=8, dim=128, page=256, blocks=1, causal=True),          # many pieces
    dict(old=[700, 1], n=1, append=True, heads=12, heads_kv=4, dim=128, page=24, blocks=3, causal=True),         # an odd page
    dict(old=[500, 33, 90], n=4, append=True, heads=8, heads_kv=8, dim=64, page=40, blocks=5, causal=True),
    dict(old=[300, 40], n=2, append=True, heads=7, heads_kv=1, dim=64, page=3, blocks=3, causal=True),           # a scale per token
    dict(old=[300, 1000], n=1, append=True, heads=8, heads_kv=2, dim=128, page=64, blocks=4, causal=True, window_size=(100, 0)),
    dict(old=[90, 200], n=5, append=0, heads=4, heads_kv=2, dim=64, page=16, blocks=1, window_size=(30, 2)),
    dict(old=[90, 200], n=5, append=2, heads=4, heads_kv=2, dim=64, page=16, blocks=1, causal=True),             # fewer new tokens than queries
    dict(old=[5, 200], n=1, append=7, heads=4, heads_kv=2, dim=64, page=16, blocks=2),                           # more of them
    dict(old=[1, 2], n=9, append=0, heads=4, heads_kv=2, dim=32, page=16, blocks=1, causal=True),                # rows ahead of the sequence see nothing
    dict(old=[0, 0], n=1, append=0, heads=4, heads_kv=2, dim=32, page=16, blocks=1),                             # nothing cached
    dict(old=[400, 77], n=2, append=True, heads=4, heads_kv=2, dim=128, page=64, blocks=2, causal=True, softmax_scale=-0.11),
    dict(old=[400, 77], n=2, append=True, heads=4, heads_kv=2, dim=128, page=64, blocks=2, causal=True, num_splits=3),
    dict(old=[400, 77], n=2, append=True, heads=4, heads_kv=2, dim=128, page=500, blocks=10, causal=True, paged=False),
    dict(old=[100, 300, 9], n=1, append=True, heads=4, heads_kv=2, dim=64, page=512, blocks=4, causal=True, paged=False, rows=[3, 0, 2],
         leftpad=[0, 17, 130]),
    dict(old=[0, 300], n=3, append=True, heads=4, heads_kv=2, dim=64, page=512, blocks=4, causal=True, paged=False, leftpad=[5, 60]),
    dict(old=[17], n=33, append=True, heads=2, heads_kv=1, dim=64, page=16, blocks=1, causal=True),
    dict(old=[100, 555], n=70, append=True, heads=8, heads_kv=2, dim=128, page=64, blocks=4, causal=True),
    dict(old=[260, 0], n=130, append=True, heads=6, heads_kv=2, dim=64, page=128, blocks=1, causal=True),
    dict(old=[100, 333], n=40, append=True, heads=4, heads_kv=1, dim=256, page=32, blocks=2, causal=True),
]


@pytest.mark.parametrize("code", [INT8, E4M3], ids=["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("case", range(len(ATTENDS)))
def test_attend(case, dtype, code):
    run_attend(1000 + case, dtype=dtype, code=code, **ATTENDS[case])


CHUNKS = [
    # one query tile per CTA, then two; contiguous caches shorter than a tile of keys, rows and pads of their own
    dict(old=[20, 7], n=40, append=True, heads=4, heads_kv=2, dim=64, page=72, blocks=9, causal=True, paged=False),
    dict(old=[20, 0], n=70, append=True, heads=8, heads_kv=2, dim=128, page=96, blocks=6, causal=True, paged=False),
    dict(old=[100, 300, 9], n=70, append=True, heads=8, heads_kv=2, dim=64, page=512, blocks=32, causal=True, paged=False, rows=[3, 0, 2]),
    dict(old=[100, 300, 9], n=70, append=True, heads=8, heads_kv=2, dim=128, page=512, blocks=4, causal=True, paged=False, rows=[3, 0, 2],
         leftpad=[0, 17, 130]),
    # rows ahead of the sequence see nothing
    dict(old=[10, 45], n=40, append=0, heads=4, heads_kv=2, dim=64, page=16, blocks=1, causal=True),
    dict(old=[10, 85, 0], n=80, append=0, heads=8, heads_kv=2, dim=128, page=16, blocks=1, causal=True),
    dict(old=[0, 0], n=80, append=0, heads=8, heads_kv=2, dim=64, page=16, blocks=1),
    # windows, to the right too
    dict(old=[200, 90], n=40, append=0, heads=4, heads_kv=2, dim=128, page=32, blocks=2, window_size=(30, 2)),
    dict(old=[400, 290], n=90, append=True, heads=8, heads_kv=2, dim=64, page=32, blocks=2, window_size=(100, 3)),
    dict(old=[700, 290], n=90, append=True, heads=8, heads_kv=2, dim=128, page=128, blocks=1, causal=True, window_size=(150, 0)),
    # no mask, keys past the last one in the tile; groups that are no power of two; a scale per key; a scale of 0
    dict(old=[129, 383], n=65, append=True, heads=6, heads_kv=2, dim=64, page=48, blocks=3),
    dict(old=[250, 31], n=200, append=True, heads=3, heads_kv=1, dim=128, page=80, blocks=5, causal=True),
    dict(old=[100], n=50, append=True, heads=4, heads_kv=1, dim=256, page=16, blocks=16, causal=True),
    dict(old=[100, 600], n=70, append=True, heads=4, heads_kv=1, dim=64, page=16, blocks=1, causal=True, softmax_scale=0.0),
    # few units: keys in pieces
    dict(old=[3000], n=33, append=True, heads=4, heads_kv=1, dim=64, page=64, blocks=4, causal=True),
    dict(old=[2500, 100], n=33, append=True, heads=8, heads_kv=1, dim=128, page=256, blocks=2, causal=True),
    dict(old=[1500], n=20, append=True, heads=1, heads_kv=1, dim=256, page=128, blocks=1, causal=True),
]


@pytest.mark.parametrize("code", [INT8, E4M3], ids=["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("case", range(len(CHUNKS)))
def test_attend_chunks(case, dtype, code):
    run_attend(2000 + 100 * case, dtype=dtype, code=code, **CHUNKS[case])


@pytest.mark.parametrize("n,heads", [(1, 4), (30, 4), (90, 8)])
def test_attend_large_scores(n, heads):
    """Scores up to 60: the maximum moves a lot, and one key takes nearly all."""
    run_attend(9, [300, 70], n, True, heads, 2, 64, 16, 1, F16, INT8, causal=True, q_gain=15.0)


@pytest.mark.parametrize("n", [1, 40])
def test_attend_alibi(n):
    slopes = torch.tensor([[0.5, 0.1, 0.03, 0.0], [0.2, 0.2, 0.01, 1.0]], device=DEV)
    run_attend(7, [300, 80], n, True, 4, 2, 64, 16, 1, BF16, E4M3, causal=True, alibi_slopes=slopes)


def test_attend_hidden_scales_do_not_reach_a_row():
    """Blocks of NaN or infinite scale behind a window, and codes of NaN behind the end of a sequence, leave the outputs alone."""
    page, B, n, heads, dim = 16, 2, 2, 4, 64
    old = [100, 61]
    table, pool = make_table(3, old, page)
    kc, ks = make_cache(31, pool, page, 2, dim, E4M3, 1)
    vc, vs = make_cache(32, pool, page, 2, dim, E4M3, 1)
    q = rand(33, B, n, heads, dim).to(F16)
    # keys from len - n - 40 on are seen: whole pages before that
    for b, length in enumerate(old):
        for p in range((length - n - 40) // page):
            ks[table[b, p]], vs[table[b, p]] = math.nan, math.inf
        tail = length % page
        kc.view(torch.int8)[table[b, length // page], tail:] = 0x7f
        vc.view(torch.int8)[table[b, length // page], tail:] = 0x7f
    want, weight = ref.attend(q, ref.values(kc, ks), ref.values(vc, vs), old, causal=True, window=(40, 0), table=table)
    out = fa().flash_attn_with_kvcache(q.to(DEV), kc.to(DEV), vc.to(DEV), cache_seqlens=torch.tensor(old, device=DEV), block_table=table.to(DEV),
                                       causal=True, window_size=(40, 0), k_scale=ks.to(DEV), v_scale=vs.to(DEV)).double().cpu()
    assert ((out - want).abs() <= ref.tolerance(want, weight, F16, 100, 10.0)).all()


def rotated(x, positions, cos, sin, interleaved):
    """Rotary embedding of x (batch, tokens, heads, dim), every product and sum rounded to its type."""
    n = cos.shape[1] * 2
    c, s = cos[positions][:, :, None], sin[positions][:, :, None]
    part, rest = x[..., :n], x[..., n:]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else part.chunk(2, -1)
    ra, rb = a * c - b * s, a * s + b * c
    out = torch.stack([ra, rb], -1).flatten(-2) if interleaved else torch.cat([ra, rb], -1)
    return torch.cat([out, rest], -1)


@pytest.mark.parametrize("code", [INT8, E4M3], ids=["int8", "e4m3"])
@pytest.mark.parametrize("interleaved,share", [(True, 1.0), (False, 1.0), (False, 0.5)])
@pytest.mark.parametrize("n,heads,dim,dtype", [(1, 8, 128, BF16), (3, 4, 64, F16), (20, 8, 128, BF16), (90, 8, 64, F16), (25, 4, 256, BF16)])
def test_attend_rotary(n, heads, dim, dtype, interleaved, share, code):
    """New keys are rotated before they are quantised, the queries as they are read; scales and caches with strides of their own."""
    page, old, hk = 32, [45, 130], 2
    table, pool = make_table(6, [x + n for x in old], page)
    kc, ks = make_cache(61, pool, page, hk, dim, code, 2)
    vc, vs = make_cache(62, pool, page, hk, dim, code, 2)
    both = torch.stack([ref.bits(kc), ref.bits(vc)], 2).to(DEV).view(code)          # (pages, page, 2, heads, dim)
    scales = torch.stack([ks, vs]).permute(0, 3, 1, 2).contiguous().to(DEV).permute(0, 2, 3, 1)
    qkv = rand(63, 2, n, heads + 2 * hk, dim).to(dtype)
    q, k, v = qkv.split([heads, hk, hk], 2)
    angle = rand(64, 240, int(dim * share) // 2)
    cos, sin = torch.cos(angle).to(dtype), torch.sin(angle).to(dtype)
    dq, dk, dv = qkv.to(DEV).split([heads, hk, hk], 2)
    out = fa().flash_attn_with_kvcache(dq, both[:, :, 0], both[:, :, 1], dk, dv, cos.to(DEV), sin.to(DEV), cache_seqlens=torch.tensor(old, device=DEV),
                                       block_table=table.to(DEV), causal=True, rotary_interleaved=interleaved, k_scale=scales[0], v_scale=scales[1])
    at = torch.tensor(old)[:, None] + torch.arange(n)
    ref.append_call(rotated(k, at, cos, sin, interleaved), kc, ks, old, table=table)
    ref.append_call(v, vc, vs, old, table=table)
    same_cache(both[:, :, 0].contiguous(), kc)
    same_cache(both[:, :, 1].contiguous(), vc)
    assert torch.equal(scales[0].cpu(), ks) and torch.equal(scales[1].cpu(), vs)
    vv = ref.values(vc, vs)
    want, weight = ref.attend(rotated(q, at, cos, sin, interleaved), ref.values(kc, ks), vv, [x + n for x in old], causal=True, table=table)
    assert ((out.double().cpu() - want).abs() <= ref.tolerance(want, weight, dtype, 220, float(vv.abs().max()))).all()


@pytest.mark.parametrize("n,heads,dim,blocks", [(1, 2, 64, 1), (40, 4, 64, 1), (90, 8, 128, 1), (24, 4, 256, 1), (40, 4, 64, 2)])
def test_attend_scales_that_are_no_numbers(n, heads, dim, blocks):
    """Rows that see a block of NaN or infinite scale are no numbers; rows that do not (before it, or past it by the window) are as without
    it, and so are rows in front of codes of NaN behind the end."""
    page, old, hk = 16, [160 + n, 75 + n], 2
    table, pool = make_table(7, old, page)
    for spoil_v in (False, True):
        kc, ks = make_cache(71, pool, page, hk, dim, E4M3, blocks)
        vc, vs = make_cache(72, pool, page, hk, dim, E4M3, blocks)
        q = rand(73, 2, n, heads, dim).to(F16)
        (vs if spoil_v else ks)[table[0, 5], 0, 0] = math.inf if spoil_v else math.nan    # keys 80 on of sequence 0, head 0
        for b, length in enumerate(old):
            if length % page:
                kc.view(torch.int8)[table[b, length // page], length % page:] = 0x7f
                vc.view(torch.int8)[table[b, length // page], length % page:] = 0x7f
        clean_k, clean_v = ks.nan_to_num(0.01), torch.where(torch.isfinite(vs), vs, 0.01)
        for window in ((-1, -1), (60, 0)):
            want, weight = ref.attend(q, ref.values(kc, clean_k).nan_to_num(), ref.values(vc, clean_v).nan_to_num(), old, causal=True, window=window,
                                      table=table)
            out = fa().flash_attn_with_kvcache(q.to(DEV), kc.to(DEV), vc.to(DEV), cache_seqlens=torch.tensor(old, device=DEV), block_table=table.to(DEV),
                                               causal=True, window_size=window, k_scale=ks.to(DEV), v_scale=vs.to(DEV)).double().cpu()
            rows = 16 // blocks
            at = torch.arange(old[0] - n, old[0])
            sees = (at >= 80) & ((at - window[0] < 80 + rows) if window[0] >= 0 else True)
            spoilt = torch.zeros(2, n, heads, dtype=torch.bool)
            spoilt[0, :, :heads // hk] = sees[:, None]
            fine = ((out - want).abs() <= ref.tolerance(want, weight, F16, 300, 10.0)).all(-1)
            assert fine[~spoilt].all()
            assert not torch.isfinite(out[spoilt]).any()


@pytest.mark.parametrize("batch,n,dim", [(600, 1, 64), (600, 2, 32), (40, 20, 64), (33, 70, 128)])
def test_attend_large_batches(batch, n, dim):
    run_attend(8, [(37 * i) % 70 for i in range(batch)], n, True, 4, 2, dim, 16, 1, BF16, E4M3, causal=True)


def test_offsets_past_32_bits():
    """Pages beyond 4 GiB of codes: tables, append, a decode step and chunks."""
    page, heads, dim, blocks = 256, 8, 256, 4
    pages = 9000                                       # 4.7e9 codes in each cache
    kc = torch.empty(pages, page, heads, dim, dtype=torch.int8, device=DEV)
    vc = torch.empty_like(kc)
    ks, vs = (torch.full((pages, blocks, heads), float("nan"), device=DEV) for _ in range(2))
    table = torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    free = torch.tensor([8999, 4095, 8192, 8191, 8900], dtype=torch.int32, device=DEV)
    lens = [300, 77]
    slots, _, used = fa().build_block_table(torch.zeros(2, device=DEV), torch.tensor(lens, device=DEV), free, table, page, sum(lens))
    assert int(used) == 3 and slots.max().item() > 2 ** 21
    k, v = rand(81, sum(lens), heads, dim).to(BF16), rand(82, sum(lens), heads, dim).to(BF16)
    fa().kvcache_append(k.to(DEV), v.to(DEV), kc, vc, slots, ks, vs)
    small = torch.tensor([[0, 1, 4], [2, 3, 4]])       # the same pages of a small cache
    p_kc, p_vc = (torch.zeros(5, page, heads, dim, dtype=torch.int8) for _ in range(2))
    p_ks, p_vs = (torch.full((5, blocks, heads), float("nan")) for _ in range(2))
    at = torch.cat([torch.arange(300), 2 * page + torch.arange(77)])
    ref.append_slots(k, p_kc, p_ks, at)
    ref.append_slots(v, p_vc, p_vs, at)
    order = table[:, :2].flatten().long().cpu()[[0, 1, 2]]
    assert torch.equal(kc[order.to(DEV)].cpu()[0], p_kc[0]) and torch.equal(ks[order.to(DEV)].cpu()[:2, 0], p_ks[:2, 0])
    table[1, 1:], table[0, 2] = 8191, 8900
    for n in (1, 20, 150):
        q = rand(83 + n, 2, n, 16, dim).to(BF16)
        kn, vn = rand(84 + n, 2, n, heads, dim).to(BF16), rand(85 + n, 2, n, heads, dim).to(BF16)
        out = fa().flash_attn_with_kvcache(q.to(DEV), kc, vc, kn.to(DEV), vn.to(DEV), cache_seqlens=torch.tensor(lens, device=DEV), block_table=table,
                                           causal=True, k_scale=ks, v_scale=vs)
        place = dict(table=small)
        ref.append_call(kn, p_kc, p_ks, lens, **place)
        ref.append_call(vn, p_vc, p_vs, lens, **place)
        lens = [x + n for x in lens]
        vv = ref.values(p_vc, p_vs)
        want, weight = ref.attend(q, ref.values(p_kc, p_ks), vv, lens, causal=True, **place)
        assert ((out.double().cpu() - want).abs() <= ref.tolerance(want, weight, BF16, max(lens), 4.0)).all()


def test_chunks_stay_off_after_a_wait_ran_out():
    from flash_attn_triton_b200 import _native as N
    kc, ks = (t.to(DEV) for t in make_cache(95, 4, 64, 2, 64, INT8, 1))
    q = torch.zeros(1, 40, 4, 64, dtype=F16, device=DEV)
    call = lambda q: fa().flash_attn_with_kvcache(q, kc, kc, cache_seqlens=torch.tensor([50], device=DEV), cache_batch_idx=torch.zeros(1, device=DEV),
                                                  k_scale=ks, v_scale=ks)
    dev = torch.cuda.current_device()
    assert N.lib().fa_debug_set_wait_status(dev, 31) == 0
    try:
        with pytest.raises(N.DeviceWaitError):
            call(q)
        call(q[:, :1])                                 # decode waits for nothing
    finally:
        assert N.lib().fa_device_wait_clear(dev) == 0
    call(q)


def test_attend_scales_far_apart():
    """Blocks whose scales differ by 2^30: what a row sees of small values, where its weight is on them, keeps its precision."""
    page, dim = 16, 64
    old = [64]
    table, pool = make_table(4, old, page)
    kc, ks = make_cache(41, pool, page, 1, dim, INT8, 1)
    vc, vs = make_cache(42, pool, page, 1, dim, INT8, 1)
    q = rand(43, 1, 1, 2, dim)
    vs[table[0, 0]] *= 2.0 ** 30
    ks[table[0, 0]] *= 0.0                            # score 0; the other blocks' scores are pushed up or far below
    vs[table[0, 2]] = 0.0                             # a block of zeros
    for sign in (1.0, -1.0):
        kc2 = kc.clone()
        kc2[table[0, 1]] = (sign * 127 * torch.sign(q[0, 0, :1])).to(torch.int8)
        qh = (q * 6).to(F16)
        want, weight = ref.attend(qh, ref.values(kc2, ks), ref.values(vc, vs), old, table=table)
        out = fa().flash_attn_with_kvcache(qh.to(DEV), kc2.to(DEV), vc.to(DEV), cache_seqlens=torch.tensor(old, device=DEV),
                                           block_table=table.to(DEV), k_scale=ks.to(DEV), v_scale=vs.to(DEV)).double().cpu()
        # p_j is rounded against the largest p_j v_j; the output against fp16's range
        fits = want.abs() < 65504
        tol = ref.tolerance(want, weight, F16, 64, float((weight.max())))
        assert ((out - want).abs() <= tol)[fits].all()


def test_attend_queries_of_any_magnitude():
    """bf16 queries are brought into the range of fp16: as precise at 2^-60 and 2^60 as at 1 when the scale undoes it."""
    page, dim, old = 16, 64, [200]
    table, pool = make_table(5, old, page)
    kc, ks = make_cache(51, pool, page, 1, dim, INT8, 1)
    vc, vs = make_cache(52, pool, page, 1, dim, INT8, 1)
    q = rand(53, 1, 1, 4, dim).to(BF16)
    q[0, 0, 3] = 0
    outs = []
    for e in (0, -60, 60):
        outs.append(fa().flash_attn_with_kvcache((q * 2.0 ** e).to(DEV), kc.to(DEV), vc.to(DEV), cache_seqlens=torch.tensor(old, device=DEV),
                                                 block_table=table.to(DEV), softmax_scale=0.125 * 2.0 ** -e, k_scale=ks.to(DEV),
                                                 v_scale=vs.to(DEV)))
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


# ---- block tables ------------------------------------------------------------------------------------------------------
TABLES = [
    # old, new, page
    ([0], [1], 16),
    ([16, 15, 17, 0], [1, 1, 1, 0], 16),
    ([0, 5, 100, 31], [700, 0, 28, 1], 32),
    ([3, 3, 3], [5, 6, 7], 1),
    ([7] * 300, [(i * 7919) % 40 for i in range(300)], 24),
    ([0, 9] * 1000, [1, 3] * 1000, 48),
    ([0, 100000], [200000, 1], 4096),
]


@pytest.mark.parametrize("case", range(len(TABLES)))
@pytest.mark.parametrize("padding", [0, 1, 1000])
def test_block_table(case, padding):
    old, new, page = TABLES[case]
    have, need = [-(-n // page) for n in old], [-(-(n + m) // page) for n, m in zip(old, new)]
    rng = np.random.default_rng(case)
    order = rng.permutation(sum(need) + 5).astype(np.int32)
    wide = torch.full((len(old), max(need) + 7), -3, dtype=torch.int32)
    table = wide[:, 2:-3]                              # a slice: rows of another pitch
    at = 0
    for b, n in enumerate(have):
        table[b, :n] = torch.from_numpy(order[at:at + n])
        at += n
    free = torch.from_numpy(order[at:])
    want, slots, cu, used = wide.clone(), [], [0], 0
    rows = want[:, 2:-3]
    for b, (n, m) in enumerate(zip(old, new)):
        for p in range(have[b], need[b]):
            rows[b, p] = free[used]
            used += 1
        slots += [int(rows[b, p // page]) * page + p % page for p in range(n, n + m)]
        cu.append(len(slots))
    total = len(slots) + padding
    got = wide.to(DEV)
    g_slots, g_cu, g_used = fa().build_block_table(torch.tensor(old, device=DEV), torch.tensor(new, device=DEV, dtype=torch.int32), free.to(DEV),
                                                   got[:, 2:-3], page, total)
    assert g_slots.dtype == torch.int64 and g_cu.dtype == torch.int32 and g_used.dtype == torch.int32
    assert g_slots.tolist() == slots + [-1] * padding and g_cu.tolist() == cu and int(g_used) == used
    assert torch.equal(got.cpu(), want)


def test_block_table_of_no_requests():
    e = torch.empty(0, dtype=torch.int32, device=DEV)
    slots, cu, used = fa().build_block_table(e, e, e, torch.empty(0, 4, dtype=torch.int32, device=DEV), 16, 3)
    assert slots.tolist() == [-1, -1, -1] and cu.tolist() == [0] and int(used) == 0


BAD_TABLES = [
    ([-1, 3], [1, 1], 8, 10, 100, "negative"),
    ([1, 3], [1, -1], 8, 10, 100, "negative"),
    ([1, 3], [60, 60], 8, 100, 119, "num_tokens"),
    ([1, 3], [60, 1], 8, 6, 100, "too few pages"),
    ([1, 250], [1, 7], 8, 100, 100, "exceeds its row"),
    ([2 ** 31 - 1, 0], [2 ** 31 - 1, 0], 1, 100, 100, "num_tokens"),
]


@pytest.mark.parametrize("case", range(len(BAD_TABLES)))
def test_block_table_refusals(case):
    old, new, page, pages, slots, message = BAD_TABLES[case]
    table = torch.full((2, 32), 7, dtype=torch.int32, device=DEV)
    args = (torch.tensor(old, device=DEV, dtype=torch.int32), torch.tensor(new, device=DEV, dtype=torch.int32),
            torch.arange(pages, dtype=torch.int32, device=DEV), table, page, slots)
    with pytest.raises(ValueError, match=message):
        fa().build_block_table(*args)
    assert (table == 7).all()
    fa().set_validation(False)
    try:
        s, cu, used = fa().build_block_table(*args)
    finally:
        fa().set_validation(True)
    assert (s == -1).all() and (cu == 0).all() and int(used) == -1 and (table == 7).all()


# ---- refusals ------------------------------------------------------------------------------------------------------------
def test_append_refusals_write_nothing():
    page, heads, dim, pool = 16, 2, 64, 4
    for tokens in (20, 6000):                          # checks by one CTA, and by a grid of them
        big = max(pool, -(-tokens // page) + 1)
        kc, ks = make_cache(60, big, page, heads, dim, INT8, 2)
        x = rand(61, tokens, heads, dim).to(F16).to(DEV)
        good = torch.arange(tokens)
        behind, twice, again = good.clone(), good.clone(), good.clone()
        behind[-1] = big * page
        twice[-1] = twice[-2]
        again[1] = tokens - 1                          # into the block of the last tokens
        for slots, message in ((behind, "behind the cache"), (twice, "returns to a block"), (again, "returns to a block")):
            kd, vd, ksd, vsd = kc.to(DEV), kc.to(DEV), ks.to(DEV), ks.to(DEV)
            with pytest.raises(ValueError, match=message):
                fa().kvcache_append(x, x, kd, vd, slots.to(DEV), ksd, vsd)
            assert torch.equal(kd.cpu(), kc) and torch.equal(vd.cpu(), kc) and torch.equal(ksd.cpu(), ks) and torch.equal(vsd.cpu(), ks)
        fa().set_validation(False)
        try:                                           # a slot behind the cache is passed over
            kd, vd, ksd, vsd = kc.to(DEV), kc.to(DEV), ks.to(DEV), ks.to(DEV)
            fa().kvcache_append(x, x, kd, vd, behind.to(DEV), ksd, vsd)
        finally:
            fa().set_validation(True)
        want, wants = kc.clone(), ks.clone()
        ref.append_slots(x.cpu(), want, wants, torch.cat([good[:-1], torch.tensor([-1])]))
        assert torch.equal(kd.cpu(), want) and torch.equal(ksd.cpu(), wants)


def test_attend_refusals_write_nothing():
    page, heads, dim, pool = 16, 2, 64, 6
    kc, ks = make_cache(62, pool, page, heads, dim, INT8, 1)
    q = rand(63, 2, 1, heads, dim).to(F16).to(DEV)
    for wide in (3, 600):                              # tables checked by every CTA, and by a kernel of their own
        table = torch.zeros(2, wide, dtype=torch.int32)
        table[1] = 1
        for lens, bad_page, message in (([5, 40], pool, "physical page"), ([5, wide * page], 0, "do not fit"), ([-1, 5], 0, "do not fit")):
            t = table.clone()
            t[1, 1] = bad_page
            kd, vd, ksd, vsd = kc.to(DEV), kc.to(DEV), ks.to(DEV), ks.to(DEV)
            with pytest.raises(ValueError, match=message):
                fa().flash_attn_with_kvcache(q, kd, vd, q, q, cache_seqlens=torch.tensor(lens, device=DEV), block_table=t.to(DEV), k_scale=ksd,
                                             v_scale=vsd)
            assert torch.equal(kd.cpu(), kc) and torch.equal(vd.cpu(), kc) and torch.equal(ksd.cpu(), ks) and torch.equal(vsd.cpu(), ks)


def test_argument_refusals():
    mk = lambda *s, dtype=torch.int8: torch.zeros(*s, dtype=dtype, device=DEV)
    q, cache, scale = mk(1, 1, 2, 64, dtype=F16), mk(4, 16, 2, 64), mk(4, 2, 2, dtype=torch.float32)
    call = lambda **kw: fa().flash_attn_with_kvcache(**{**dict(q=q, k_cache=cache, v_cache=cache.clone(), cache_seqlens=3,
                                                             cache_batch_idx=torch.zeros(1, device=DEV), k_scale=scale, v_scale=scale.clone()), **kw})
    call()
    for kw, message in ((dict(k_scale=None), "need k_scale"), (dict(k_scale=scale.half()), "float32"), (dict(k_scale=scale[:3]), "shape"),
                        (dict(k_scale=scale[:, :1]), "shape"), (dict(k_scale=mk(4, 3, 2, dtype=torch.float32), v_scale=mk(4, 3, 2, dtype=torch.float32)), "divide"),
                        (dict(k_cache=cache.view(E4M3)), "both"), (dict(k_cache=cache.half(), v_cache=cache.half()), "go with"),
                        (dict(q=q.float()), "FP16 and BF16"), (dict(k=cache[:1, :1], v=cache[:1, :1]), "same dtype"),
                        (dict(k_cache=mk(4, 16, 2, 72)[..., 4:68]), "aligned")):
        with pytest.raises(ValueError, match=message):
            call(**kw)
    with pytest.raises(ValueError, match="1 to 1024"):
        call(k_cache=mk(1, 2048, 2, 64), v_cache=mk(1, 2048, 2, 64), k_scale=mk(1, 1, 2, dtype=torch.float32), v_scale=mk(1, 1, 2, dtype=torch.float32))
    k = mk(5, 2, 64, dtype=F16)
    app = lambda **kw: fa().kvcache_append(**{**dict(k=k, v=k, k_cache=cache, v_cache=cache.clone(), slot_mapping=torch.arange(5, device=DEV), k_scale=scale,
                                                     v_scale=scale.clone()), **kw})
    app()
    for kw, message in ((dict(k=k[0]), "shape"), (dict(v=k[:4]), "shape"), (dict(k=k.float(), v=k.float()), "FP16 or BF16"),
                        (dict(slot_mapping=torch.arange(4, device=DEV)), "one integer slot"), (dict(slot_mapping=torch.arange(5.0, device=DEV)), "one integer slot"),
                        (dict(k=mk(5, 3, 64, dtype=F16), v=mk(5, 3, 64, dtype=F16)), "incompatible"), (dict(k=k.cpu(), v=k.cpu()), "CUDA")):
        with pytest.raises(ValueError, match=message):
            app(**kw)
    table, n = mk(2, 4, dtype=torch.int32), torch.ones(2, dtype=torch.int32, device=DEV)
    build = lambda **kw: fa().build_block_table(**{**dict(cache_seqlens=n, new_lens=n, free_pages=torch.arange(4, device=DEV), block_table=table, page_size=16,
                                                          num_tokens=2), **kw})
    build()
    for kw, message in ((dict(block_table=table.long()), "int32"), (dict(block_table=table.cpu()), "CUDA"), (dict(block_table=table.T), "unit stride"),
                        (dict(block_table=table[:1].expand(2, -1)), "overlap"), (dict(page_size=0), "positive"), (dict(num_tokens=-1), "non-negative"),
                        (dict(num_tokens=2 ** 31), "below"), (dict(new_lens=n[:1]), "one length")):
        with pytest.raises(ValueError, match=message):
            build(**kw)


def test_append_of_nothing():
    cache, scale = torch.zeros(2, 16, 2, 64, dtype=torch.int8, device=DEV), torch.zeros(2, 1, 2, device=DEV)
    k = torch.zeros(0, 2, 64, dtype=F16, device=DEV)
    fa().kvcache_append(k, k, cache, cache.clone(), torch.zeros(0, dtype=torch.int64, device=DEV), scale, scale.clone())
    q = torch.zeros(0, 1, 2, 64, dtype=F16, device=DEV)
    out = fa().flash_attn_with_kvcache(q, cache, cache, cache_seqlens=torch.zeros(0, dtype=torch.int32, device=DEV),
                                       block_table=torch.zeros(0, 1, dtype=torch.int32, device=DEV), k_scale=scale, v_scale=scale)
    assert out.shape == q.shape


# ---- together --------------------------------------------------------------------------------------------------------------
class Server:
    """A pool of pages and requests that grow, as a serving loop keeps them; `plain` mirrors the cache on the CPU."""

    def __init__(self, seed, requests, pages, page, blocks, heads, heads_kv, dim, dtype, code, most):
        self.page, self.heads, self.heads_kv, self.dim, self.dtype = page, heads, heads_kv, dim, dtype
        self.seed, self.lens = seed, [0] * requests
        self.kc = torch.zeros(pages, page, heads_kv, dim, dtype=torch.int8, device=DEV).view(code)
        self.vc = self.kc.clone()
        self.ks = torch.full((pages, blocks, heads_kv), float("nan"), device=DEV)       # nothing is read that was not written
        self.vs = self.ks.clone()
        self.free = torch.from_numpy(np.random.default_rng(seed).permutation(pages).astype(np.int32)).to(DEV)
        self.table = torch.zeros(requests, most, dtype=torch.int32, device=DEV)
        self.plain = [t.cpu() for t in (self.kc, self.vc, self.ks, self.vs)]

    def tokens(self, n, heads):
        self.seed += 1
        return rand(self.seed, n, heads, self.dim).to(self.dtype)

    def prompts(self, new, padding):
        slots, cu, used = fa().build_block_table(torch.tensor(self.lens, device=DEV), torch.tensor(new, device=DEV), self.free, self.table, self.page,
                                                 sum(new) + padding)
        self.free = self.free[int(used):]
        k, v = self.tokens(sum(new) + padding, self.heads_kv), self.tokens(sum(new) + padding, self.heads_kv)
        fa().kvcache_append(k.to(DEV), v.to(DEV), self.kc, self.vc, slots, self.ks, self.vs)
        ref.append_slots(k, self.plain[0], self.plain[2], slots.cpu())
        ref.append_slots(v, self.plain[1], self.plain[3], slots.cpu())
        self.lens = [a + b for a, b in zip(self.lens, new)]

    def step(self, n):
        B = len(self.lens)
        _, _, used = fa().build_block_table(torch.tensor(self.lens, device=DEV), torch.full((B,), n, device=DEV), self.free, self.table, self.page, B * n)
        self.free = self.free[int(used):]
        q = self.tokens(B * n, self.heads).view(B, n, self.heads, self.dim)
        k, v = (self.tokens(B * n, self.heads_kv).view(B, n, self.heads_kv, self.dim) for _ in range(2))
        out = fa().flash_attn_with_kvcache(q.to(DEV), self.kc, self.vc, k.to(DEV), v.to(DEV), cache_seqlens=torch.tensor(self.lens, device=DEV),
                                           block_table=self.table, causal=True, k_scale=self.ks, v_scale=self.vs)
        place = dict(table=self.table.cpu())
        ref.append_call(k, self.plain[0], self.plain[2], self.lens, **place)
        ref.append_call(v, self.plain[1], self.plain[3], self.lens, **place)
        self.lens = [x + n for x in self.lens]
        vv = ref.values(self.plain[1], self.plain[3])
        want, weight = ref.attend(q, ref.values(self.plain[0], self.plain[2]), vv, self.lens, causal=True, **place)
        tol = ref.tolerance(want, weight, self.dtype, max(self.lens), float(vv.nan_to_num().abs().max()))
        assert ((out.double().cpu() - want).abs() <= tol).all()

    def check(self):
        same_cache(self.kc, self.plain[0])
        same_cache(self.vc, self.plain[1])
        assert torch.equal(self.ks.cpu().nan_to_num(-1), self.plain[2].nan_to_num(-1))
        assert torch.equal(self.vs.cpu().nan_to_num(-1), self.plain[3].nan_to_num(-1))


@pytest.mark.parametrize("code", [INT8, E4M3], ids=["int8", "e4m3"])
@pytest.mark.parametrize("page,blocks,dim,dtype", [(16, 1, 64, BF16), (48, 3, 128, F16)])
def test_serving_loop(page, blocks, dim, dtype, code):
    s = Server(70, 5, 120, page, blocks, 8, 2, dim, dtype, code, 30)
    s.prompts([17, 160, 0, 1, 64], 13)
    s.step(1)
    s.step(1)
    s.prompts([0, 33, 90, 0, 2], 0)
    s.step(3)
    s.step(40)
    s.step(1)
    s.check()


def test_captured_step():
    """Tables, append and attention of a decode step captured once and replayed as the requests grow, beside eager calls."""
    page, B, dim, pages = 16, 3, 64, 64
    lens = torch.tensor([5, 15, 30], dtype=torch.int32, device=DEV)
    one = torch.ones(B, dtype=torch.int32, device=DEV)
    free = torch.arange(pages - 1, 7, -1, dtype=torch.int32, device=DEV)
    table = torch.zeros(B, 8, dtype=torch.int32, device=DEV)
    table[0, 0], table[1, 0], table[2, :2] = 1, 2, torch.tensor([3, 4], dtype=torch.int32, device=DEV)
    kc, ks = (t.to(DEV) for t in make_cache(80, pages, page, 2, dim, INT8, 1))
    vc, vs = (t.to(DEV) for t in make_cache(81, pages, page, 2, dim, INT8, 1))
    start = [t.clone() for t in (kc, vc, ks, vs, table)]
    q, k, v = (torch.zeros(B, 1, h, dim, dtype=BF16, device=DEV) for h in (8, 2, 2))

    def step():
        slots, _, used = fa().build_block_table(lens, one, free, table, page, B + 2)
        pad = torch.zeros(2, 2, dim, dtype=BF16, device=DEV)
        fa().kvcache_append(torch.cat([k.flatten(0, 1), pad]), torch.cat([v.flatten(0, 1), pad]), kc, vc, slots, ks, vs)
        out = fa().flash_attn_with_kvcache(q, kc, vc, cache_seqlens=lens + 1, block_table=table, causal=True, k_scale=ks, v_scale=vs)
        both = fa().flash_attn_with_kvcache(q, kc, vc, k, v, cache_seqlens=lens + 1, block_table=table, causal=True, k_scale=ks, v_scale=vs)
        return out, both, used

    fa().set_validation(False)
    try:
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = step()
        for t, s in zip((kc, vc, ks, vs, table), start):
            t.copy_(s)
        seen = []
        for i in range(20):
            for t, seed in ((q, 1), (k, 2), (v, 3)):
                t.copy_(rand(1000 * i + seed, *t.shape))
            graph.replay()
            seen.append([x.clone() for x in captured])
            free_used = int(captured[2])
            free.copy_(torch.cat([free[free_used:], free[:free_used]]))
            lens.add_(1)
        end = [t.clone() for t in (kc, vc, ks, vs, table)]
        # the same eagerly
        for t, s in zip((kc, vc, ks, vs, table), start):
            t.copy_(s)
        lens.copy_(torch.tensor([5, 15, 30]))
        free.copy_(torch.arange(pages - 1, 7, -1))
        for i in range(20):
            for t, seed in ((q, 1), (k, 2), (v, 3)):
                t.copy_(rand(1000 * i + seed, *t.shape))
            now = step()
            assert all(torch.equal(a, b) for a, b in zip(now, seen[i])), i
            free.copy_(torch.cat([free[int(now[2]):], free[:int(now[2])]]))
            lens.add_(1)
        assert all(torch.equal(a, b) for a, b in zip((kc, vc, ks, vs, table), end))
    finally:
        fa().set_validation(True)


def test_streams_and_threads():
    """Calls on streams and threads of their own, each with its caches, at once: as alone."""
    import threading
    page, dim, old = 16, 64, [900, 100]
    table, pool = make_table(90, [n + 8 for n in old], page)
    sets = []
    for i in range(4):
        kc, ks = make_cache(91 + 2 * i, pool, page, 2, dim, E4M3, 1)
        sets.append([t.to(DEV) for t in (rand(95 + i, 2, 1, 16, dim).to(F16), kc, kc.clone(), rand(99 + i, 2, 1, 2, dim).to(F16), ks, ks.clone())])
    lens, tab = torch.tensor(old, dtype=torch.int32, device=DEV), table.to(DEV)

    def call(q, kc, vc, k, ks, vs):
        out = []
        for _ in range(20):
            out.append(fa().flash_attn_with_kvcache(q, kc, vc, k, k, cache_seqlens=lens, block_table=tab, causal=True, k_scale=ks, v_scale=vs))
        return out

    alone = [call(*[t.clone() for t in s]) for s in sets]
    got, errors = [None] * 4, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                got[i] = call(*sets[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:                         # noqa: BLE001 (reported below)
            errors.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors
    for a, b in zip(alone, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
