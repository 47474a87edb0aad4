"""Performance cases of serving from a paged KV cache held in 8 bits.

A case is a dict of plain values.  Its `kind` picks the operator:

  tables   build_block_table          pages for the new tokens of every request, their slots, cu_seqlens
  append   kvcache_append             packed new keys and values into the 8-bit cache, by slot
  attend   flash_attn_with_kvcache    (append to and) attend to the 8-bit cache, int8 or e4m3 codes

A cache holds codes (pages, page_size, heads_kv, dim) and one fp32 scale per block of `block` tokens and head, (pages,
page_size / block, heads_kv); a value is code * scale.  The first token of a block starts its scale afresh; a later token
that is larger than the scale allows raises it, and the codes that the block keeps are rounded again to the new one.

With `own` false run() computes the same in elementary torch operations, in 32 bits.  Lengths belong to the case
(`lens_seed`), the values of the tensors to the seed of prepare().
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
_LARGEST = {"int8": 127.0, "e4m3": 448.0}


def _tables(name, **kw):
    # `share` of the requests bring a prompt of up to `longest_new` tokens, the others one token
    c = dict(name=name, kind="tables", requests=8, longest=4096, share=0.0, longest_new=1, page=16, padding=0, lens_seed=1)
    c.update(kw)
    return c


def _append(name, **kw):
    c = dict(name=name, kind="append", dtype="bf16", code="e4m3", requests=24, shortest=17, longest=2048, cached=0, heads_kv=8,
             dim=128, page=64, block=64, lens_seed=2)
    c.update(kw)
    return c


def _attend(name, **kw):
    c = dict(name=name, kind="attend", dtype="bf16", code="e4m3", batch=64, shortest=1024, longest=32768, tokens=1, append=True,
             heads=32, heads_kv=8, dim=128, page=256, block=256, window=-1, lens_seed=3)
    c.update(kw)
    return c


def listed():
    return [
        # a decode step of a handful of conversations: latency
        _tables("tables_decode"),
        # continuous batching: most requests decode, some bring a chunk of their prompt, the slots padded to a fixed size
        _tables("tables_mixed", requests=301, longest=20000, share=0.1, longest_new=2048, padding=777, lens_seed=4),
        # a large offline batch of prompts
        _tables("tables_prompts", requests=2048, longest=64, share=1.0, longest_new=2048, lens_seed=5),
        # one new token of each of a few requests, most of them into blocks that hold tokens already
        _append("append_decode", dtype="fp16", code="int8", requests=32, shortest=1, longest=1, cached=3000, heads_kv=4, dim=64, page=16,
                block=16),
        # prompts of very different lengths
        _append("append_ragged"),
        # prompt processing of a large batch
        _append("append_prompts", code="int8", requests=64, shortest=1024, longest=8192, cached=100, page=256, block=32, lens_seed=6),
        # one decode step of a single conversation: latency
        _attend("attend_single", batch=1, shortest=1900, longest=1900, page=16, block=16),
        # one decode step of a large batch with long contexts
        _attend("attend_batch", dtype="fp16", code="int8"),
        # four drafted tokens of each request verified at once; narrow heads, an odd page
        _attend("attend_drafts", batch=16, shortest=300, longest=4000, tokens=4, heads=16, heads_kv=4, dim=64, page=48, block=16,
                lens_seed=7),
        # a decode step over long caches with a sliding window and wide heads
        _attend("attend_window", code="int8", batch=20, shortest=500, longest=20000, heads=16, heads_kv=4, dim=256, page=128, block=64,
                window=4095, lens_seed=8),
        # a chunk of each of four prompts behind what is cached of them
        _attend("attend_chunk", batch=4, shortest=1024, longest=8192, tokens=256, page=64, block=64, lens_seed=9),
        # the last, odd chunk of two long prompts
        _attend("attend_prompt", dtype="fp16", code="int8", batch=2, shortest=5000, longest=11000, tokens=1537, page=16, block=16,
                lens_seed=10),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("tables", "append", "append", "attend", "attend", "attend"))
    c = None
    while c is None or _cost(c) > _LIMIT[kind]:
        page = rng.choice((16, 16, 24, 32, 48, 64, 128, 256))
        block = rng.choice([b for b in (8, 16, 32, 64, 128, 256) if page % b == 0])
        common = dict(dtype=rng.choice(("fp16", "bf16")), code=rng.choice(("int8", "e4m3")), dim=rng.choice((64, 128, 128, 256)),
                      heads_kv=rng.choice((1, 2, 4, 8)), page=page, block=block, lens_seed=rng.randrange(1 << 20))
        if kind == "tables":
            c = _tables("", requests=_log_int(rng, 1, 2048), longest=_log_int(rng, 1, 20000), share=rng.choice((0.0, 0.1, 1.0)),
                        longest_new=_log_int(rng, 1, 2048), page=page, padding=rng.choice((0, 0, _log_int(rng, 1, 5000))),
                        lens_seed=common["lens_seed"])
        elif kind == "append":
            longest = rng.choice((1, 1, _log_int(rng, 2, 8192)))
            c = _append("", requests=_log_int(rng, 1, 128), shortest=max(1, longest // rng.choice((1, 8, 64))), longest=longest,
                        cached=rng.choice((0, _log_int(rng, 1, 4000))), **common)
        else:
            longest = _log_int(rng, 64, 32768)
            tokens = rng.choice((1, 1, 1, rng.choice((2, 3, 4, 8)), _log_int(rng, 16, 2048)))
            c = _attend("", batch=_log_int(rng, 1, 64), shortest=max(1, longest // rng.choice((1, 4, 32))), longest=longest, tokens=tokens,
                        append=rng.random() < 0.8, heads=common["heads_kv"] * rng.choice((1, 4, 8)),
                        window=rng.choice((-1, -1, -1, _log_int(rng, 128, 8192))), **common)
    del c["name"]
    return c


# the most one drawn case of a kind may cost, in the units of _cost: below the largest listed one
_LIMIT = {"tables": 17e6, "append": 0.7e9, "attend": 1.2e9}


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 200) * (4 if c.get("tokens", 1) > 64 else 1)


def _lens(c):
    """(tokens cached, new tokens) of every request, as numpy arrays."""
    rng = np.random.default_rng(c["lens_seed"])
    if c["kind"] == "tables":
        n = c["requests"]
        new = np.where(rng.random(n) < c["share"], rng.integers(1, c["longest_new"] + 1, n), 1)
        return rng.integers(0, c["longest"] + 1, n), new
    if c["kind"] == "append":
        n = c["requests"]
        new = rng.integers(c["shortest"], c["longest"] + 1, n)
        return rng.integers(0, c["cached"] + 1, n), new
    old = rng.integers(c["shortest"], c["longest"] + 1, c["batch"])
    return old, np.full(c["batch"], c["tokens"])


def _pages(c, lens):
    """Block table of requests of these lengths, from a shuffled pool with some pages to spare, and the pool's size.  A row
    ends in copies of its first page."""
    need = -(-lens // c["page"])
    pool = int(need.sum()) + 8
    order = np.random.default_rng(c["lens_seed"] + 1).permutation(pool).astype(np.int32)
    table = np.zeros((len(lens), int(need.max())), dtype=np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        table[b, n:] = order[at]
        at += n
    return table, pool


def _values(gen, dtype, *shape):
    """Keys or values as projections give them: unit variance, a few channels much larger."""
    x = torch.randn(*shape, device="cuda", generator=gen)
    x *= 1 + 5 * (torch.rand(shape[-1], device="cuda", generator=gen) < 0.03)
    return x.to(dtype)


def _cache(gen, c, pool):
    """Codes and scales of a cache in use."""
    shape = (pool, c["page"], c["heads_kv"], c["dim"])
    x = torch.randn(*shape, device="cuda", dtype=torch.float16, generator=gen)
    x.mul_(_LARGEST[c["code"]] / 4).clamp_(-_LARGEST[c["code"]], _LARGEST[c["code"]])
    codes = x.round_().to(torch.int8) if c["code"] == "int8" else x.to(torch.float8_e4m3fn)
    del x
    scales = torch.rand(pool, c["page"] // c["block"], c["heads_kv"], device="cuda", generator=gen)
    return codes, (0.5 + scales) * (4 / _LARGEST[c["code"]])


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    old, new = _lens(c)
    s = dict(case=c, cache_seqlens=torch.tensor(old, dtype=torch.int32, device="cuda"))
    if c["kind"] == "tables":
        have, need = -(-old // c["page"]), -(-(old + new) // c["page"])
        pool = int(need.sum()) + 64
        order = torch.randperm(pool, device="cuda", generator=gen).to(torch.int32)
        table = torch.zeros(len(old), int(need.max()) + 3, dtype=torch.int32, device="cuda")
        filled = torch.arange(table.shape[1], device="cuda") < torch.tensor(have, device="cuda")[:, None]
        table[filled] = order[:int(have.sum())]
        s.update(table=table, free=order[int(have.sum()):].contiguous(), slots=int(new.sum()) + c["padding"],
                 new_lens=torch.tensor(new, dtype=torch.int32, device="cuda"))
        return s
    table, pool = _pages(c, old + new)
    dt = _DTYPES[c["dtype"]]
    s["k_cache"], s["k_scale"] = _cache(gen, c, pool)
    s["v_cache"], s["v_scale"] = _cache(gen, c, pool)
    if c["kind"] == "append":
        at = np.concatenate([np.arange(n, n + m) for n, m in zip(old, new)])
        seq = np.repeat(np.arange(len(old)), new)
        slots = table[seq, at // c["page"]].astype(np.int64) * c["page"] + at % c["page"]
        s["slots"] = torch.from_numpy(slots).cuda()
        s["k"], s["v"] = (_values(gen, dt, len(slots), c["heads_kv"], c["dim"]) for _ in range(2))
        return s
    s["table"] = torch.from_numpy(table).cuda()
    s["q"] = _values(gen, dt, c["batch"], c["tokens"], c["heads"], c["dim"])
    s["k"] = s["v"] = None
    if c["append"]:
        s["k"], s["v"] = (_values(gen, dt, c["batch"], c["tokens"], c["heads_kv"], c["dim"]) for _ in range(2))
    else:
        s["cache_seqlens"] += c["tokens"]
    return s


def _plain_tables(cached, new, free, table, page, slots):
    have, need = (cached + page - 1) // page, (cached + new + page - 1) // page
    first = torch.cumsum(need - have, 0) - (need - have)
    cu = torch.cat([new.new_zeros(1), torch.cumsum(new, 0, dtype=torch.int32)])
    column = torch.arange(table.shape[1], device=table.device)[None, :]
    fresh = (column >= have[:, None]) & (column < need[:, None])
    taken = free[(first[:, None] + column - have[:, None]).clamp(0, free.numel() - 1)]
    table.copy_(torch.where(fresh, taken, table))
    t = torch.arange(slots, device=table.device)
    seq = torch.searchsorted(cu[1:], t, right=True).clamp(max=cached.numel() - 1)
    pos = cached[seq] + t - cu[seq]
    block = table[seq, (pos // page).clamp(max=table.shape[1] - 1)].long()
    slot = torch.where(t < cu[-1], block * page + pos % page, -1)
    return table, slot, cu, (need - have).sum(dtype=torch.int32)


def _coded(x, code):
    """Nearest code of each value."""
    x = x.clamp(-_LARGEST[code], _LARGEST[code])
    return x.round().to(torch.int8) if code == "int8" else x.to(torch.float8_e4m3fn)


def _plain_append(x, slots, cache, scale, code):
    """x (tokens, heads, dim) into the cache, in place."""
    rows = cache.shape[1] // scale.shape[1]              # tokens of a block
    codes, scales = cache.view(-1, rows, *cache.shape[2:]), scale.view(-1, scale.shape[2])
    x = x.float()
    block, row = slots // rows, slots % rows
    starts = torch.cat([block.new_ones(1, dtype=torch.bool), block[1:] != block[:-1]])
    group = torch.cumsum(starts, 0) - 1                  # the tokens of one block are neighbours
    touched, kept = block[starts], row[starts]           # tokens that a block keeps
    largest = torch.zeros(touched.numel(), x.shape[1], device=x.device)
    largest.scatter_reduce_(0, group[:, None].expand(-1, x.shape[1]), x.abs().amax(-1), "amax")
    old = torch.where(kept[:, None] > 0, scales[touched], 0.0)
    need = largest / torch.tensor(_LARGEST[code], device=x.device)
    now = torch.maximum(old, torch.where(need < torch.finfo(torch.float32).tiny, 0.0, need))
    inverse = torch.where(now > 0, 1 / now, 0.0)
    again = (kept > 0) & (now > old).any(-1)             # a scale is raised over codes that stay
    at = touched[again]
    held = codes[at]
    moved = _coded(held.float() * (old * inverse)[again][:, None, :, None], code)
    stays = torch.arange(rows, device=x.device) < kept[again][:, None]
    raised = (now > old)[again]
    bits = torch.where((stays[:, :, None] & raised[:, None, :])[..., None], moved.view(torch.int8), held.view(torch.int8))
    codes.view(torch.int8)[at] = bits
    codes.view(torch.int8)[block, row] = _coded(x * inverse[group][..., None], code).view(torch.int8)
    scales[touched] = now


def _positions(cached, tokens, capacity):
    return (cached[:, None] + torch.arange(tokens, device=cached.device)).clamp(max=capacity - 1)


def _plain_attend(q, k_cache, v_cache, k_scale, v_scale, table, lens, window):
    """q (batch, tokens, heads, dim) are the last tokens of sequences of `lens` tokens; causal."""
    batch, tokens, heads, dim = q.shape
    pages, page, heads_kv, _ = k_cache.shape
    rows = page // k_scale.shape[1]

    def gathered(cache, scale):
        x = cache.view(pages, -1, rows, heads_kv, dim)[table].float() * scale[table][:, :, :, None, :, None]
        return x.view(batch, -1, heads_kv, dim)

    k, v = gathered(k_cache, k_scale), gathered(v_cache, v_scale)
    q = q.float().view(batch, tokens, heads_kv, heads // heads_kv, dim)
    scores = torch.einsum("bthgd,bkhd->bhgtk", q, k) / math.sqrt(dim)
    del k
    key = torch.arange(scores.shape[-1], device=q.device)
    at = lens[:, None] - tokens + torch.arange(tokens, device=q.device)
    hidden = key > at[..., None]
    if window >= 0:
        hidden |= key < at[..., None] - window
    scores.masked_fill_(hidden[:, None, None], float("-inf"))
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1).permute(0, 3, 1, 2)
    return (torch.einsum("bhgtk,bkhd->bthgd", scores, v) / total[..., None]).reshape(batch, tokens, heads, dim)


def run(state):
    s, c = state, state["case"]
    if c["kind"] == "tables":
        if own:
            import flash_attn_triton_b200 as fa
            slots, cu, used = fa.build_block_table(s["cache_seqlens"], s["new_lens"], s["free"], s["table"], c["page"], s["slots"])
            return s["table"], slots, cu, used
        return _plain_tables(s["cache_seqlens"], s["new_lens"], s["free"], s["table"], c["page"], s["slots"])
    cache = s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]
    if c["kind"] == "append":
        if own:
            import flash_attn_triton_b200 as fa
            fa.kvcache_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], k_scale=s["k_scale"], v_scale=s["v_scale"])
            return cache
        _plain_append(s["k"], s["slots"], s["k_cache"], s["k_scale"], c["code"])
        _plain_append(s["v"], s["slots"], s["v_cache"], s["v_scale"], c["code"])
        return cache
    window = (c["window"], 0) if c["window"] >= 0 else (-1, -1)
    if own:
        import flash_attn_triton_b200 as fa
        out = fa.flash_attn_with_kvcache(s["q"], s["k_cache"], s["v_cache"], s["k"], s["v"], cache_seqlens=s["cache_seqlens"],
                                         block_table=s["table"], causal=True, window_size=window, k_scale=s["k_scale"],
                                         v_scale=s["v_scale"])
        return (out, *cache) if c["append"] else (out,)
    lens = s["cache_seqlens"]
    if c["append"]:
        at = _positions(lens, c["tokens"], s["table"].shape[1] * c["page"])
        slots = (torch.gather(s["table"].long(), 1, at // c["page"]) * c["page"] + at % c["page"]).flatten()
        _plain_append(s["k"].flatten(0, 1), slots, s["k_cache"], s["k_scale"], c["code"])
        _plain_append(s["v"].flatten(0, 1), slots, s["v_cache"], s["v_scale"], c["code"])
        lens = lens + c["tokens"]
    out = _plain_attend(s["q"], *cache, s["table"], lens, c["window"]).to(s["q"].dtype)
    return (out, *cache) if c["append"] else (out,)


def work(case):
    """Bytes: what is read, once, and what is written, once.  Operations: two products per visible pair of an attention, and a
    few per element that is quantised or entry that is built."""
    c = case
    old, new = _lens(c)
    if c["kind"] == "tables":
        have, need = -(-old // c["page"]), -(-(old + new) // c["page"])
        tokens, taken = int(new.sum()), int((need - have).sum())
        partly = int((old % c["page"] != 0).sum())       # pages that hold tokens already and take more
        slots = tokens + c["padding"]
        return {"bytes": 8.0 * len(old) + 4.0 * (2 * taken + partly) + 8.0 * slots + 4.0 * (len(old) + 2), "flops": 10.0 * slots}
    H, D = c["heads_kv"], c["dim"]
    tokens, blocks = int(new.sum()), int((-(-(old + new) // c["block"]) - old // c["block"]).sum())
    appended = 2.0 * tokens * H * D * (2 + 1) + 2 * 4.0 * blocks * H
    if c["kind"] == "append":
        return {"bytes": appended + 8.0 * tokens + 4.0 * 2 * H * int((old % c["block"] != 0).sum()), "flops": 6.0 * tokens * H * D}
    first = np.maximum(old - c["window"], 0) if c["window"] >= 0 else 0 * old
    seen = old + new - first if not c["append"] else old - first
    pairs = 0
    for n in old.tolist():
        at = np.arange(n, n + c["tokens"], dtype=np.int64)
        pairs += int((at - (np.maximum(at - c["window"], 0) if c["window"] >= 0 else 0) + 1).sum())
    codes = 2.0 * int(seen.sum()) * H * D + 2 * 4.0 * H * int((-(-seen // c["block"])).sum())
    q = 2 * 2.0 * c["batch"] * c["tokens"] * c["heads"] * D
    return {"bytes": codes + q + (appended if c["append"] else 0.0), "flops": 4.0 * D * c["heads"] * pairs}


# ---- the same in 64 bits, request by request ---------------------------------------------------------------------------
def _exact_append(x, where, cache, scale, code):
    """Rows x (tokens, heads, dim) of one request, at slots `where` (a list), into the cache."""
    block_rows = cache.shape[1] // scale.shape[1]
    flat_codes, flat_scales = cache.view(-1, *cache.shape[2:]), scale.view(-1, scale.shape[2])
    at = 0
    while at < len(where):
        block = where[at] // block_rows
        end = at
        while end < len(where) and where[end] // block_rows == block:
            end += 1
        kept = where[at] % block_rows
        rows = x[at:end].double()
        before = flat_scales[block].double()
        need = rows.abs().amax(dim=(0, 2)) / _LARGEST[code]
        after = torch.maximum(before, need) if kept else need
        after = after.float().double()
        safe = torch.where(after == 0, 1.0, after)
        if kept:
            held = flat_codes[block * block_rows:block * block_rows + kept]
            grown = (after > before)[None, :, None]
            fitted = _coded((held.double() * (before / safe)[None, :, None]).float(), code)
            held.view(torch.int8).copy_(torch.where(grown, fitted.view(torch.int8), held.view(torch.int8)))
        first = block * block_rows + kept
        flat_codes[first:first + end - at] = _coded((rows / safe[None, :, None]).float(), code)
        flat_scales[block] = after.float()
        at = end


def exact(case, seed):
    """Scales and attention outputs from their definition in 64 bits; whole numbers and codes have none.  None where the walk over
    the blocks would take long."""
    c = case
    if c["kind"] == "tables":
        return None
    old, new = _lens(c)
    append = c["kind"] == "append" or c["append"]
    if append and int((new // c["block"] + 2).sum()) > 6000:
        return None
    s = prepare(case, seed)
    table, _ = _pages(c, old + new)
    start = 0
    for b, (n, m) in enumerate(zip(old.tolist(), new.tolist())):
        if not append:
            break
        where = [int(table[b, p // c["page"]]) * c["page"] + p % c["page"] for p in range(n, n + m)]
        for name in ("k", "v"):
            rows = s[name][start:start + m] if c["kind"] == "append" else s[name][b]
            _exact_append(rows, where, s[name + "_cache"], s[name + "_scale"], c["code"])
        start += m
    scales = (None, None, s["k_scale"].double(), s["v_scale"].double())
    if c["kind"] == "append":
        return scales
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    group, block = c["heads"] // c["heads_kv"], c["block"]
    for b, n in enumerate((old + new).tolist()):
        low = max(0, n - c["tokens"] - c["window"]) if c["window"] >= 0 else 0
        pos = torch.arange(low, n, device="cuda")
        page, row = s["table"][b].long()[pos // c["page"]], pos % c["page"]
        queries = torch.arange(n - c["tokens"], n, device="cuda")
        ahead = pos[None, :] > queries[:, None]
        if c["window"] >= 0:
            ahead |= pos[None, :] < queries[:, None] - c["window"]
        for h in range(c["heads_kv"]):
            k = s["k_cache"][page, row, h].double() * s["k_scale"][page, row // block, h].double()[:, None]
            v = s["v_cache"][page, row, h].double() * s["v_scale"][page, row // block, h].double()[:, None]
            for g in range(h * group, (h + 1) * group):
                logits = (s["q"][b, :, g].double() @ k.T) * c["dim"] ** -0.5
                out[b, :, g] = torch.softmax(logits.masked_fill(ahead, -math.inf), dim=-1) @ v
    return (out, *scales) if c["append"] else (out,)
