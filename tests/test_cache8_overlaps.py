"""Calls that append to the 8-bit KV cache write codes and scales of keys and values: arrays that overlap are refused on the host."""
import ctypes
import itertools
import random

import pytest
from test_cache8_refusals import append, cache, decode, native  # noqa: F401 (native: a fixture)

PAGES, PAGE, HEADS, DIM = 4, 64, 2, 128
K, V, KS, VS = 1 << 20, 1 << 24, 1 << 28, 1 << 29
CODES, SCALES = (PAGE * HEADS * DIM, HEADS * DIM, DIM), (4 * HEADS, HEADS, 1)         # packed


def refused(N, k=K, v=V, k_stride=CODES, v_stride=CODES, ks=KS, vs=VS, ks_stride=SCALES, vs_stride=SCALES, pages=PAGES, blocks=4, heads=HEADS, dim=DIM):
    """By all calls alike; those that are not refused for this want a workspace, and launch nothing."""
    c = cache(N, block=PAGE // blocks, k_scale=ks, v_scale=vs, ks_stride=N._I64x3(*ks_stride), vs_stride=N._I64x3(*vs_stride))
    place = dict(page_size=PAGE, num_pages=pages, head_dim=dim, k_cache=k, v_cache=v, kc_stride=N._I64x3(*k_stride), vc_stride=N._I64x3(*v_stride))
    a = append(N, cache=c, heads=heads, **place)
    d = decode(N, heads_kv=heads, heads_q=heads, k_new=4096, v_new=4096, seqlen_new=1, kn_stride=N._I64x3(1024, 1024, 128),
               vn_stride=N._I64x3(1024, 1024, 128), **place)
    failed, lib = ctypes.c_uint32(), N.lib()
    calls = [lambda: lib.fa_append8_checked(ctypes.byref(a), ctypes.byref(failed), None),
             lambda: lib.fa_decode_paged8(ctypes.byref(d), ctypes.byref(c), None),
             lambda: lib.fa_decode_paged8_checked(ctypes.byref(d), ctypes.byref(c), ctypes.byref(failed), None)]
    got = []
    for call in calls:
        status = call()
        assert status < 0
        got.append(status == -1 and "must not overlap" in lib.fa_last_error().decode())
        assert got[-1] or status != -1, lib.fa_last_error()
    assert len(set(got)) == 1
    return got[0]


def test_layouts(native):
    N = native
    assert not refused(N)
    wide = tuple(2 * s for s in CODES[:2]) + (DIM,)
    assert not refused(N, v=K + HEADS * DIM, k_stride=wide, v_stride=wide)                       # (pages, page, 2, heads, dim)
    halves = (2 * CODES[0],) + CODES[1:]
    assert not refused(N, v=K + CODES[0], k_stride=halves, v_stride=halves)                      # (pages, 2, page, heads, dim)
    assert not refused(N, v=K + CODES[0], k_stride=halves, v_stride=(halves[0], DIM, PAGE * DIM))  # one of them by heads
    assert not refused(N, k_stride=(CODES[0], DIM, PAGE * DIM), v_stride=(DIM, PAGES * HEADS * DIM, PAGES * DIM))
    for kw in (dict(v=K), dict(v=K + 16), dict(v=K + CODES[0]), dict(v=K + 3 * CODES[0] + CODES[1]), dict(k_stride=(0,) + CODES[1:]),
               dict(v_stride=CODES[:2] + (0,)), dict(k_stride=(CODES[0], DIM, DIM)), dict(v=K + HEADS * DIM - 16, k_stride=wide, v_stride=wide)):
        assert refused(N, **kw), kw
    assert not refused(N, v=K + PAGES * CODES[0]) and not refused(N, v=K - PAGES * CODES[0])
    assert not refused(N, ks_stride=(1, 4 * HEADS, 4), vs_stride=(4, 16, 64))
    assert not refused(N, vs=KS + 4, ks_stride=(16, 4, 2), vs_stride=(16, 4, 2)) and not refused(N, vs=KS + 4 * PAGES * 8)
    for kw in (dict(vs=KS), dict(vs=KS + 4), dict(ks_stride=(8, 0, 1)), dict(vs_stride=(0, 2, 1)), dict(ks_stride=(0, 0, 0)), dict(vs_stride=(8, 2, 2)),
               dict(vs=KS + 4 * 31), dict(vs=KS + 8, ks_stride=(16, 4, 2), vs_stride=(16, 4, 2))):
        assert refused(N, **kw), kw
    # one page, one block, one head: their strides are nothing
    one = dict(pages=1, blocks=1, heads=1, k_stride=(0, DIM, 0), v_stride=(16, DIM, 16), ks_stride=(0, 0, 0), vs_stride=(1, 1, 1))
    assert not refused(N, **one)
    assert refused(N, **{**one, "vs": KS}) and refused(N, **{**one, "v": K + DIM})


def test_reading_calls_take_them(native):
    N = native
    d = decode(N, k_cache=K, v_cache=K, kc_stride=N._I64x3(0, HEADS * DIM, DIM), vc_stride=N._I64x3(0, HEADS * DIM, DIM))
    c = cache(N, k_scale=KS, v_scale=KS)                                                         # strides of 0
    assert native.lib().fa_decode_paged8(ctypes.byref(d), ctypes.byref(c), None) != -1


@pytest.mark.parametrize("seed", range(3))
def test_against_counting(native, seed):
    """Random strides and distances: whatever shares a word is refused, and where the strides nest and are the same, nothing else is."""
    rng = random.Random(seed)
    seen = set()
    for _ in range(1500):
        pages, blocks, heads = rng.randint(1, 4), rng.choice((1, 2, 4)), rng.randint(1, 3)
        sizes = (pages, blocks, heads)

        def nested():
            order, stride, reach = rng.sample(range(3), 3), [0, 0, 0], 1
            for d in order:
                stride[d] = reach + rng.choice((0, 0, 1, reach))
                reach += (sizes[d] - 1) * stride[d]
            return stride
        kind = rng.randrange(3)
        ks = [rng.randint(-3, 20) for _ in range(3)] if kind == 0 else nested()
        vs = list(ks) if kind == 1 else nested()
        delta = rng.randint(-70, 70)
        words = lambda s: [sum(i * t for i, t in zip(at, s)) for at in itertools.product(*map(range, sizes))]
        k, v = words(ks), [delta + x for x in words(vs)]
        shared = len(set(k)) < len(k) or len(set(v)) < len(v) or bool(set(k) & set(v))
        got = refused(native, vs=KS + 4 * delta, ks_stride=ks, vs_stride=vs, pages=pages, blocks=blocks, heads=heads,
                      k_stride=(heads * DIM * PAGE, heads * DIM, DIM), v_stride=(heads * DIM * PAGE, heads * DIM, DIM))
        assert got or not shared, (sizes, ks, vs, delta)
        if kind == 1:
            assert got == shared, (sizes, ks, vs, delta)
        seen.add((kind, shared, got))
    assert {(1, True, True), (1, False, False), (0, True, True), (2, False, False)} <= seen
