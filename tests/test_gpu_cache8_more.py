"""KV cache in 8 bits, beside test_gpu_cache8.py: many pieces of one sequence, tokens that are no numbers, scales
far apart in chunks, negative scales."""
import math

import pytest
import torch

import cache8_reference as ref
from test_gpu_cache8 import BF16, E4M3, F16, INT8, fa, make_cache, make_table, rand, run_attend, same_cache
from util import DEV

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("old", [74000, 131040])
@pytest.mark.parametrize("dim,dtype,code", [(64, F16, E4M3), (128, BF16, INT8)])
def test_chunk_of_one_unit_behind_a_long_context(dim, dtype, code, old):
    """One KV head, one pair of query tiles: more pieces asked for than a merge has room for.  The call after it is not refused."""
    from flash_attn_triton_b200 import _native as N
    run_attend(11, [old], 32, True, 8, 1, dim, 256, 1, dtype, code, causal=True)
    torch.cuda.synchronize()
    assert N.lib().fa_device_wait_status(torch.cuda.current_device()) == 0
    run_attend(12, [100], 32, True, 8, 1, dim, 256, 1, dtype, code, causal=True)


@pytest.mark.parametrize("code", [INT8, E4M3], ids=["int8", "e4m3"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_append_writes_no_codes_of_nan(bad, code):
    """Tokens that are no numbers: codes of 0 under a scale of NaN or infinity, by slot, for blocks that one lane holds and larger ones;
    tokens that come behind them too, until the block is started again."""
    for page, dim in ((16, 32), (1024, 64)):
        kc, ks = make_cache(21, 2, page, 2, dim, code, 1)
        x = rand(22, page - 4, 2, dim).to(BF16)
        x[3, 1, 5] = bad
        kd, vd, ksd, vsd = kc.to(DEV), kc.to(DEV), ks.to(DEV), ks.to(DEV)
        fa().kvcache_append(x.to(DEV), x.to(DEV), kd, vd, torch.arange(page, 2 * page - 4, device=DEV), ksd, vsd)
        more = rand(23, 2, 2, dim).to(BF16)
        fa().kvcache_append(more.to(DEV), more.to(DEV), kd, vd, torch.arange(2 * page - 4, 2 * page - 2, device=DEV), ksd, vsd)
        for codes, scale in ((kd, ksd), (vd, vsd)):
            codes, scale = codes.cpu(), scale.cpu()
            assert (ref.bits(codes)[1, :page - 2, 1] == 0).all() and not math.isfinite(scale[1, 0, 1])
            assert ref.values(codes, scale)[1, :page - 2, 1].isnan().all() and torch.isfinite(ref.values(codes, scale)[1, :page - 2, 0]).all()
            assert torch.equal(ref.bits(codes)[0], ref.bits(kc)[0])


SPOILT = [
    # query tokens, heads, dim, page, blocks: decode, one query tile per CTA, two; a scale per key (blocks of 4)
    (3, 4, 64, 16, 1),
    (8, 4, 256, 32, 2),
    (40, 4, 64, 16, 1),
    (40, 4, 128, 16, 4),
    (40, 4, 256, 16, 1),
    (100, 8, 64, 16, 1),
    (100, 8, 128, 32, 2),
]


@pytest.mark.parametrize("code", [INT8, E4M3], ids=["int8", "e4m3"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("new", [False, True], ids=["cached", "new"])
@pytest.mark.parametrize("case", range(len(SPOILT)))
def test_tokens_that_are_no_numbers_spoil_the_rows_that_see_them(case, new, bad, code):
    """A NaN or infinity among the cached values, whose block the window of most rows has passed, or among the new ones, where earlier
    rows do not see its block: those rows, in one tile of keys with it, are as without it."""
    n, heads, dim, page, blocks = SPOILT[case]
    hk, size = 2, page // blocks
    first = 208 if new else 100 // size * size         # of the block
    old = [208 - min(8, n // 2), 61]
    window = (-1, -1) if new else (94 if n <= 8 else 100, 0)
    table, pool = make_table(31, [x + n for x in old], page)
    k, v = (rand(32 + i, 2, old[0] + n, hk, dim).to(F16) for i in range(2))
    clean = v.clone()
    v[0, first + 1, 0, 3] = bad
    slots = torch.cat([torch.tensor([int(table[b, p // page]) * page + p % page for p in range(old[b])]) for b in range(2)])
    cached = lambda x: torch.cat([x[b, :old[b]] for b in range(2)])
    added = lambda x: torch.stack([x[b, old[b]:old[b] + n] for b in range(2)])
    q = rand(34, 2, n, heads, dim).to(F16)
    kc, vc = (torch.zeros(pool, page, hk, dim, dtype=torch.int8, device=DEV).view(code) for _ in range(2))
    ks, vs = (torch.zeros(pool, blocks, hk, device=DEV) for _ in range(2))
    fa().kvcache_append(cached(k).to(DEV), cached(v).to(DEV), kc, vc, slots.to(DEV), ks, vs)
    out = fa().flash_attn_with_kvcache(q.to(DEV), kc, vc, added(k).to(DEV), added(v).to(DEV), cache_seqlens=torch.tensor(old, device=DEV),
                                       block_table=table.to(DEV), causal=True, window_size=window, k_scale=ks, v_scale=vs).double().cpu()
    # with a number in that place
    pk, pv = (torch.zeros(pool, page, hk, dim, dtype=torch.int8).view(code) for _ in range(2))
    pks, pvs = torch.zeros(pool, blocks, hk), torch.zeros(pool, blocks, hk)
    for x, codes, scale in ((k, pk, pks), (clean, pv, pvs)):
        ref.append_slots(cached(x), codes, scale, slots)
        ref.append_call(added(x), codes, scale, old, table=table)
    lens = [x + n for x in old]
    want, weight = ref.attend(q, ref.values(pk, pks), ref.values(pv, pvs), lens, causal=True, window=window, table=table)
    at = torch.arange(old[0], lens[0])
    sees = (at >= first) & ((at - window[0] < first + size) if window[0] >= 0 else True)
    spoilt = torch.zeros(2, n, heads, dtype=torch.bool)
    spoilt[0, :, :heads // hk] = sees[:, None]
    assert (~sees).any() and (sees.any() or not new)
    fine = ((out - want).abs() <= ref.tolerance(want, weight, F16, max(lens), 10.0)).all(-1)
    assert fine[~spoilt].all()
    assert not torch.isfinite(out[spoilt]).any()


@pytest.mark.parametrize("code", [INT8, E4M3], ids=["int8", "e4m3"])
@pytest.mark.parametrize("n,heads,dim,blocks,leftpad", [(40, 4, 64, 16, 0), (40, 4, 128, 4, 0), (30, 4, 256, 2, 0), (40, 4, 64, 1, 5), (100, 8, 128, 16, 0),
                                                        (40, 4, 64, 1, 0), (100, 8, 64, 1, 0)])
def test_chunk_with_scales_far_apart(n, heads, dim, blocks, leftpad, code):
    """Keys whose scales of V are 2^30 above their neighbours', hidden from the earlier rows of the chunk: what those rows see keeps its
    precision."""
    page, hk = 16, 2
    size, old = page // blocks, [160, 75]              # lengths that include the chunk
    paged = leftpad == 0
    table, pool = make_table(41, old, page)
    if not paged:
        table, pool, page, blocks = None, 2, 192, 12   # the same 16 keys per scale, but not in line with tiles of 16
    place = dict(table=table) if paged else dict(leftpad=torch.tensor([leftpad, 0]))
    kc, ks = make_cache(42, pool, page, hk, dim, code, blocks)
    vc, vs = make_cache(43, pool, page, hk, dim, code, blocks)
    q = rand(44, 2, n, heads, dim).to(F16)
    # the block of key 140 of sequence 0 has large values
    at = 140 + leftpad
    row = (int(table[0, at // page]), at % page // (page // blocks)) if paged else (0, at // (page // blocks))
    vs[row] *= 2.0 ** 30
    first = 140 // size * size if paged else at // 16 * 16 - leftpad
    want, weight = ref.attend(q, ref.values(kc, ks), ref.values(vc, vs), old, causal=True, **place)
    d = lambda t: None if t is None else t.to(DEV)
    out = fa().flash_attn_with_kvcache(d(q), d(kc), d(vc), cache_seqlens=torch.tensor(old, device=DEV), block_table=d(table),
                                       cache_leftpad=d(place.get("leftpad")), causal=True, k_scale=d(ks), v_scale=d(vs)).double().cpu()
    sees = torch.zeros(2, n, dtype=torch.bool)
    sees[0] = torch.arange(old[0] - n, old[0]) >= first
    assert sees.any() and (~sees[0]).any()
    tol = ref.tolerance(want, weight, F16, max(old), 6.0)        # (no value of the others is above 3.5 * 1.6)
    assert ((out - want).abs() <= tol)[~sees].all()


def signs(seed, scale):
    """The scales, about half of them negative."""
    return torch.where(rand(seed, *scale.shape) < 0, -scale, scale)


@pytest.mark.parametrize("code", [INT8, E4M3], ids=["int8", "e4m3"])
@pytest.mark.parametrize("n,heads,dim,blocks,window", [(1, 4, 64, 1, -1), (4, 8, 128, 16, -1), (3, 4, 256, 1, 50), (40, 4, 64, 1, -1), (40, 4, 128, 4, -1),
                                                       (40, 4, 256, 1, 90), (100, 8, 64, 1, -1), (100, 8, 128, 1, 120)])
def test_attend_negative_scales(n, heads, dim, blocks, window, code):
    page, hk, old = 16, 2, [500, 260]                  # whole tiles of keys in front of the rows, and ones with a mask
    table, pool = make_table(51, old, page)
    kc, ks = make_cache(52, pool, page, hk, dim, code, blocks)
    vc, vs = make_cache(53, pool, page, hk, dim, code, blocks)
    ks, vs = signs(54, ks), signs(55, vs)
    q = (2 * rand(56, 2, n, heads, dim)).to(F16)
    want, weight = ref.attend(q, ref.values(kc, ks), ref.values(vc, vs), old, causal=True, window=(window, 0) if window >= 0 else (-1, -1), table=table)
    out = fa().flash_attn_with_kvcache(q.to(DEV), kc.to(DEV), vc.to(DEV), cache_seqlens=torch.tensor(old, device=DEV), block_table=table.to(DEV),
                                       causal=True, window_size=(window, 0) if window >= 0 else (-1, -1), k_scale=ks.to(DEV), v_scale=vs.to(DEV))
    assert ((out.double().cpu() - want).abs() <= ref.tolerance(want, weight, F16, max(old), 6.0)).all()


@pytest.mark.parametrize("code", [INT8, E4M3], ids=["int8", "e4m3"])
def test_append_to_blocks_of_negative_scale(code):
    """The sign stays where the magnitude does; where new tokens raise it, kept codes change sign."""
    page, dim, heads, pages = 16, 32, 4, 5
    kc, ks = make_cache(61, pages, page, heads, dim, code, 1)
    if code == INT8:
        kc[:, 3] = -128
    ks = signs(62, ks)
    assert (ks < 0).any() and (ks > 0).any()
    ks[1, 0, 0], ks[2, 0, 1] = -math.inf, 0.0
    slots = torch.tensor([p * page + r for p in range(pages) for r in range(5, 9)])
    x = rand(63, len(slots), heads, dim).to(F16)
    x[:8] *= 0.1                                       # below what the scales allow, then above
    x[12:] *= 9
    want, wants = kc.clone(), ks.clone()
    for p in range(pages):
        new = x[4 * p:4 * p + 4].float()
        for h in range(heads):
            old, need = ks[p, 0, h], new[:, h].abs().max() / torch.tensor(ref.LARGEST[code])
            now = old if old.abs() >= need else need
            inv = 1 / now if now != 0 and now.isfinite() else torch.zeros(())
            if need > old.abs():
                held = kc[p, :5, h].float()
                want[p, :5, h] = ref.coded((held.clamp(min=-127.0) if old < 0 and code == INT8 else held) * (old * inv), code)
            want[p, 5:9, h] = ref.coded(new[:, h] * inv if now.isfinite() else torch.zeros(4, dim), code)      # (0, not -0, under an infinite scale)
            wants[p, 0, h] = now
    kd, vd, ksd, vsd = kc.to(DEV), kc.to(DEV), ks.to(DEV), ks.to(DEV)
    fa().kvcache_append(x.to(DEV), x.to(DEV), kd, vd, slots.to(DEV), ksd, vsd)
    for codes, scale in ((kd, ksd), (vd, vsd)):
        assert torch.equal(ref.bits(codes.cpu()), ref.bits(want)) and torch.equal(scale.cpu(), wants)
    fine = wants.isfinite() & (wants != 0)             # and the new values are within half a step
    held, size = ref.values(want, wants)[:, 5:9], wants.abs().double()[:, :, :, None]
    half = size / 2 if code == INT8 else torch.maximum(x.double().view(pages, 4, heads, dim).abs() * 2.0 ** -4, size * 2.0 ** -10)
    err = (held - x.double().view(pages, 4, heads, dim)).abs()
    assert (err <= half * (1 + 1e-5))[fine.expand(-1, 4, -1)].all()


def test_overlapping_caches_and_scales():
    """Read, they are what they hold; calls that append refuse them and write nothing."""
    page, hk, dim, pool = 16, 2, 64, 4
    kc, ks = (t.to(DEV) for t in make_cache(71, pool, page, hk, dim, INT8, 1))
    vc, vs = kc.clone(), ks.clone()
    one = torch.full((1, 1, 1), 0.02, device=DEV).expand(pool, 1, hk)
    q = rand(72, 1, 1, 4, dim).to(F16).to(DEV)
    new = rand(73, 1, 1, hk, dim).to(F16).to(DEV)
    lens, rows = torch.tensor([7], device=DEV), torch.tensor([2], device=DEV)
    call = lambda kc=kc, vc=vc, ks=ks, vs=vs, k=None: fa().flash_attn_with_kvcache(q, kc, vc, k, k, cache_seqlens=lens, cache_batch_idx=rows, k_scale=ks,
                                                                                 v_scale=vs)
    flat = one.contiguous()
    assert torch.equal(call(ks=one, vs=one), call(ks=flat, vs=flat.clone()))
    assert torch.equal(call(vc=kc, vs=ks), call())
    before = [t.clone() for t in (kc, vc, ks, vs, one)]
    slots = torch.arange(3, device=DEV)
    packed = rand(74, 3, hk, dim).to(F16).to(DEV)
    for bad in (dict(ks=one), dict(vs=one), dict(ks=flat, vs=flat), dict(vc=kc), dict(kc=kc[:1].expand(pool, -1, -1, -1)), dict(ks=ks, vs=ks)):
        with pytest.raises(ValueError, match="must not overlap"):
            call(**bad, k=new)
        t = {**dict(kc=kc, vc=vc, ks=ks, vs=vs), **bad}
        with pytest.raises(ValueError, match="must not overlap"):
            fa().kvcache_append(packed, packed, t["kc"], t["vc"], slots, t["ks"], t["vs"])
    assert all(torch.equal(a, b) for a, b in zip((kc, vc, ks, vs, one), before))
    call(k=new)
    fa().kvcache_append(packed, packed, kc, vc, slots, ks, vs)
    assert not torch.equal(kc, before[0])


@pytest.mark.parametrize("code", [INT8, E4M3], ids=["int8", "e4m3"])
def test_append_to_blocks_of_tiny_scale(code):
    """A caller's scale below the smallest normal number counts as 0: zeros and tiny tokens get codes of 0 (not 0 times an infinite reciprocal)."""
    page, dim, heads = 16, 32, 3
    kc, ks = make_cache(81, 4, page, heads, dim, code, 1)
    ks[1, 0], ks[2, 0] = 1e-40, -1e-45
    slots = torch.tensor([p * page + r for p in (1, 2, 3) for r in (5, 6)])
    x = rand(82, 6, heads, dim).to(BF16)
    x[:4, 0], x[:4, 1] = 0.0, 1e-38
    kd, vd, ksd, vsd = kc.to(DEV), kc.to(DEV), ks.to(DEV), ks.to(DEV)
    fa().kvcache_append(x.to(DEV), x.to(DEV), kd, vd, slots.to(DEV), ksd, vsd)
    want, wants = kc.clone(), torch.where(ks.abs() < ref.TINY, 0.0, ks)
    ref.append_slots(x, want, wants, slots)
    for codes, scale in ((kd, ksd), (vd, vsd)):
        assert torch.equal(ref.bits(codes.cpu()), ref.bits(want)) and torch.equal(scale.cpu(), wants)
    assert (wants[1:3, 0, :2] == 0).all() and (want.float()[1:3, 5:7, :2] == 0).all()


def test_rows_far_apart():
    """Rows of a cache 32 GiB apart: an offset of two of them, in units of 16 bytes, passes 32 bits."""
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 80 * 2 ** 30:
        pytest.skip("needs 64 GiB")
    dim, rows, far = 256, 3, 2 ** 35
    memory = torch.empty(2 * far + 4096, dtype=torch.int8, device=DEV)
    wide = memory.as_strided((1, rows, 1, dim), (16, far, 256, 1))
    near, scale = make_cache(91, 1, rows, 1, dim, INT8, 1)
    other, oscale = make_cache(92, 1, rows, 1, dim, INT8, 1)
    wide.copy_(near)
    q = rand(93, 1, 1, 2, dim).to(F16).to(DEV)
    for spread_v in (False, True):
        pair = lambda x, y: (y, x) if spread_v else (x, y)
        outs = []
        for x in (wide, near.to(DEV)):
            k, v = pair(x, other.to(DEV))
            ks, vs = pair(scale.to(DEV), oscale.to(DEV))
            outs.append(fa().flash_attn_with_kvcache(q, k, v, cache_seqlens=torch.tensor([rows], device=DEV), k_scale=ks, v_scale=vs))
        assert torch.equal(*outs)
    del memory, wide
    torch.cuda.empty_cache()


def test_offsets_past_32_bits_all_that_is_written():
    """Pages beyond 4 GiB of codes: after a packed append and after each call, codes and scales of every page that the tables name."""
    page, heads, dim, blocks, pages = 256, 8, 256, 4, 9000     # 4.7e9 codes in each cache
    far = torch.tensor([8999, 4095, 8192, 8191, 8900])
    kc = torch.empty(pages, page, heads, dim, dtype=torch.int8, device=DEV)
    vc = torch.empty_like(kc)
    ks, vs = (torch.full((pages, blocks, heads), float("nan"), device=DEV) for _ in range(2))
    kc[far], vc[far] = 0, 0
    table, small = far[torch.tensor([[0, 1, 4], [2, 3, 4]])].to(torch.int32), torch.tensor([[0, 1, 4], [2, 3, 4]])
    plain = [torch.zeros(5, page, heads, dim, dtype=torch.int8) for _ in range(2)] + [torch.full((5, blocks, heads), float("nan")) for _ in range(2)]

    def compare():
        for got, want in zip((kc, vc, ks, vs), plain):
            assert torch.equal(got[far.to(DEV)].cpu().nan_to_num(-1) if want.is_floating_point() else got[far.to(DEV)].cpu(),
                               want.nan_to_num(-1) if want.is_floating_point() else want)

    lens = [300, 77]
    place = lambda t: torch.cat([t[b, torch.arange(n) // page].long() * page + torch.arange(n) % page for b, n in enumerate(lens)])
    slots = place(table)
    k, v = rand(101, sum(lens), heads, dim).to(BF16), rand(102, sum(lens), heads, dim).to(BF16)
    fa().kvcache_append(k.to(DEV), v.to(DEV), kc, vc, slots.to(DEV), ks, vs)
    ref.append_slots(k, plain[0], plain[2], place(small))
    ref.append_slots(v, plain[1], plain[3], place(small))
    compare()
    for n in (1, 20, 150):
        q, kn, vn = rand(103 + n, 2, n, 16, dim).to(BF16), rand(104 + n, 2, n, heads, dim).to(BF16), rand(105 + n, 2, n, heads, dim).to(BF16)
        fa().flash_attn_with_kvcache(q.to(DEV), kc, vc, kn.to(DEV), vn.to(DEV), cache_seqlens=torch.tensor(lens, device=DEV), block_table=table.to(DEV),
                                     causal=True, k_scale=ks, v_scale=vs)
        ref.append_call(kn, plain[0], plain[2], lens, table=small)
        ref.append_call(vn, plain[1], plain[3], lens, table=small)
        compare()
        lens = [x + n for x in lens]


GROUPS = [
    # query heads over KV heads that are no power of two apart, one token to more than a tile of rows
    (28, 4, 1), (28, 4, 2), (28, 4, 3), (28, 4, 30), (40, 8, 1), (40, 8, 3), (40, 8, 4), (10, 2, 27), (7, 1, 150),
    # rows around the limits of the kernels: 8, 16 and 128 per KV head
    (8, 1, 1), (9, 1, 1), (8, 1, 2), (17, 1, 1), (16, 1, 8), (43, 1, 3), (16, 2, 16), (16, 2, 17),
]


@pytest.mark.parametrize("code", [INT8, E4M3], ids=["int8", "e4m3"])
@pytest.mark.parametrize("heads,hk,n", GROUPS)
def test_attend_groups(heads, hk, n, code):
    for dim, dtype in ((64, BF16), (128, F16)):
        run_attend(heads + n, [90, 333], n, True, heads, hk, dim, 32, 2, dtype, code, causal=True)


def steps(seed, dim, heads, hk, n, old, page=32):
    """A call on caches of its own: (function of nothing -> (out, codes, scales), tensors that it reads)."""
    table, pool = make_table(seed, [x + n for x in old], page)
    kc, ks = (t.to(DEV) for t in make_cache(seed + 1, pool, page, hk, dim, E4M3, 1))
    vc, vs = (t.to(DEV) for t in make_cache(seed + 2, pool, page, hk, dim, E4M3, 1))
    start = [t.clone() for t in (kc, vc, ks, vs)]
    q, k, v = (rand(seed + 3 + i, len(old), n, h, dim).to(F16).to(DEV) for i, h in enumerate((heads, hk, hk)))
    lens, tab = torch.tensor(old, dtype=torch.int32, device=DEV), table.to(DEV)

    def call():
        for t, s in zip((kc, vc, ks, vs), start):
            t.copy_(s)
        out = fa().flash_attn_with_kvcache(q, kc, vc, k, v, cache_seqlens=lens, block_table=tab, causal=True, k_scale=ks, v_scale=vs)
        return [out, kc.view(torch.int8).clone(), vc.view(torch.int8).clone(), ks.clone(), vs.clone()]
    return call, (q, k, v)


PATHS = [(64, 8, 2, 1, [3000, 70]), (256, 4, 2, 4, [900, 900]), (64, 4, 1, 33, [3000]), (256, 2, 1, 40, [2000, 10]), (128, 8, 1, 40, [6000])]


@pytest.mark.parametrize("case", range(len(PATHS)))
def test_calls_repeat_themselves(case):
    """The same call gives the same bits, each of its pieces merged in their order whichever CTA comes last."""
    call, _ = steps(110 + 10 * case, *PATHS[case])
    first = call()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, call()))


def test_graphs_and_streams_at_once():
    """Two captured calls with pieces to merge, replayed at the same time on two streams beside eager calls: as alone."""
    made = [steps(210 + 10 * i, 64, 4, 1, 33, [3000 + 7 * i]) for i in range(2)] + [steps(240, 128, 8, 1, 40, [2500])]
    fa().set_validation(False)
    try:
        alone = [call() for call, _ in made]
        side = [torch.cuda.Stream() for _ in range(2)]
        graphs, outs = [], []
        for (call, _), stream in zip(made, side):
            with torch.cuda.stream(stream):
                call()
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                outs.append(call())
            graphs.append(g)
        torch.cuda.synchronize()
        for _ in range(20):
            for g, stream in zip(graphs, side):
                with torch.cuda.stream(stream):
                    g.replay()
            eager = made[2][0]()
        torch.cuda.synchronize()
        for got, want in zip(outs + [eager], alone):
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    finally:
        fa().set_validation(True)


@pytest.mark.parametrize("code", [INT8, E4M3], ids=["int8", "e4m3"])
@pytest.mark.parametrize("n,heads,dim,blocks", [(1, 4, 64, 1), (4, 8, 256, 1), (40, 4, 64, 1), (40, 4, 128, 4), (40, 4, 256, 1), (100, 8, 64, 1),
                                                (100, 8, 128, 1)])
def test_largest_weight_is_not_rounded(n, heads, dim, blocks, code):
    """fp16: one value in a cache of zeros, whose key has a row's largest score by up to 2^7.  Its weight is exactly 1 relative to the row's
    maximum, so the output is off by its own rounding and by fp32 (2^-15 of it, see cache8_reference.tolerance) alone.  Maxima are of
    score + log2 scale: blocks of zeros with scores of 0 have scales up to 1.6 / 0.3 = 2^2.4 of that value's, so rows of low scores may have
    one of them as the maximum, and a weight that is rounded (half a step more)."""
    page, hk, length = 16, 2, 300 + n
    table, pool = make_table(121, [length], page)
    kc, vc = (torch.zeros(pool, page, hk, dim, dtype=torch.int8).view(torch.int8) for _ in range(2))
    key = rand(122, hk, dim).sign()
    kc[table[0, 1], 4] = (64 * key).to(torch.int8)     # key 20: behind tiles of keys with scores of 0
    vc[table[0, 1], 4] = (rand(123, hk, dim) * 25).round().clamp(-100, 100).to(torch.int8)
    kc, vc = (ref.coded(x.float(), code) for x in (kc, vc))
    _, ks = make_cache(124, pool, page, hk, dim, code, blocks)
    _, vs = make_cache(125, pool, page, hk, dim, code, blocks)
    # score u of row r, head h: 0.5 to 5 in natural units, q as fp16 holds it
    u = torch.linspace(0.5, 5.0, n * heads).view(1, n, heads, 1)
    block = 4 // (page // blocks)
    unit = (64 * dim ** 0.5 * ks[table[0, 1], block])[None, None, :].repeat_interleave(heads // hk, -1)[..., None]
    q = (u * key.repeat_interleave(heads // hk, 0) / unit).to(F16)
    want, weight = ref.attend(q, ref.values(kc, ks), ref.values(vc, vs), [length], causal=True, table=table)
    out = fa().flash_attn_with_kvcache(q.to(DEV), kc.to(DEV), vc.to(DEV), cache_seqlens=torch.tensor([length], device=DEV), block_table=table.to(DEV),
                                       causal=True, k_scale=ks.to(DEV), v_scale=vs.to(DEV)).double().cpu()
    half = torch.finfo(F16).eps / 2 * want.abs() + torch.finfo(F16).smallest_normal * 2.0 ** -11
    others = vs[table[0].long()].amax(dim=(0, 1))      # of a head
    leads = u[..., 0] - 0.01 > torch.log(others / vs[table[0, 1], block])[None, None].repeat_interleave(heads // hk, -1)
    assert leads.sum() > leads.numel() // 2
    rounded = torch.where(leads, 0.0, 2.0 ** -11)[..., None]
    assert ((out - want).abs() <= half + (2.0 ** -15 + rounded) * weight).all()


@pytest.mark.parametrize("code", [INT8, E4M3], ids=["int8", "e4m3"])
@pytest.mark.parametrize("n,heads,dim", [(1, 4, 16), (1, 4, 64), (1, 8, 128), (1, 4, 256), (4, 4, 32), (4, 4, 64), (3, 4, 128), (4, 4, 256), (40, 4, 64),
                                         (100, 4, 128)])
def test_small_values_beside_a_heavy_zero(n, heads, dim, code):
    """A key of value 0 has nearly all of the weight, the others 2^-13 of it and small values: the sums are as exact as those values ask for,
    whatever a code is on the way (the tolerance of cache8_reference, whose largest value is 4)."""
    page, hk, length = 16, 1, 64 + n
    table, pool = make_table(131, [length], page)
    kc = torch.zeros(pool, page, hk, dim)
    vc = (rand(132, pool, page, hk, dim) * 2).round().clamp(-4, 4)
    heavy = int(table[0, 0]), 3
    key = rand(133, hk, dim).sign()
    kc[heavy], vc[heavy] = 64 * key, 0.0
    kc, vc = ref.coded(kc, code), ref.coded(vc, code)
    ks = vs = torch.ones(pool, 1, hk)
    q = (9.0 / (64 * dim ** 0.5) * key.expand(1, n, heads, dim)).to(F16)
    want, weight = ref.attend(q, ref.values(kc, ks), ref.values(vc, vs), [length], causal=True, table=table)
    out = fa().flash_attn_with_kvcache(q.to(DEV), kc.to(DEV), vc.to(DEV), cache_seqlens=torch.tensor([length], device=DEV), block_table=table.to(DEV),
                                       causal=True, k_scale=ks.to(DEV), v_scale=vs.to(DEV)).double().cpu()
    assert weight.max() < 0.08                         # (no more than 163 others of 2^-13 each, values up to 4)
    assert ((out - want).abs() <= ref.tolerance(want, weight, F16, length, 4.0)).all()
