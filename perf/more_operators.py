"""Performance cases of decoding with drafted tokens: a small model drafts a tree of tokens, the large one verifies all of them in one
step over its paged KV cache.

A case is a dict of plain values.  Its `kind` picks the operator:

  norm     qk_norm_rotary             RMS norm of every head's query and key, then the rotation by the token's position; with `train`
                                      the gradients too
  attend   flash_attn_with_kvcache    append the drafted tokens and attend: each sees the cached context and its ancestors (tree_mask)
  verify   verify_draft_tree          accept or reject drafted tokens by given random numbers, sample the token that follows
  compact  kvcache_compact            the accepted tokens' rows moved together, in the caches of all layers
  release  release_pages              pages that requests no longer need, back to the free list

A tree of a request has node 0, the last token that is certain, as its root; parents[i] < i, and -1 marks a node that the request does
not use.  With `own` false run() computes the same in elementary torch operations, in 32 bits (in 64 where the verification compares
and sums).  Lengths and trees belong to the case (`case_seed`), the values of the tensors to the seed of prepare().
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _norm(name, **kw):
    c = dict(name=name, kind="norm", dtype="bf16", batch=1, tokens=64, heads=32, heads_kv=8, dim=128, rotary=128, interleaved=False,
             wide=False, train=False, longest=16384, case_seed=1)
    c.update(kw)
    return c


def _attend(name, **kw):
    # page 0: a contiguous cache
    c = dict(name=name, kind="attend", dtype="bf16", batch=32, shortest=1024, longest=16384, nodes=16, share=0.8, heads=32, heads_kv=8,
             dim=128, page=64, case_seed=2)
    c.update(kw)
    return c


def _verify(name, **kw):
    # near: how close the draft's distribution is to the target's (the noise between their logits)
    c = dict(name=name, kind="verify", dtype="fp32", batch=32, nodes=16, branch=0.5, vocabulary=131072, near=0.7, case_seed=3)
    c.update(kw)
    return c


def _compact(name, **kw):
    c = dict(name=name, kind="compact", dtype="bf16", layers=16, batch=32, cached=300, nodes=16, heads_kv=8, dim=128, page=16, case_seed=4)
    c.update(kw)
    return c


def _release(name, **kw):
    # whole: the share of requests that have ended; the others give back what their drafted tokens took
    c = dict(name=name, kind="release", requests=64, longest=4096, drafted=16, whole=0.0, page=16, padding=0, case_seed=5)
    c.update(kw)
    return c


def listed():
    return [
        # queries and keys of the drafted tokens of 16 conversations, at the positions of their depths: latency
        _norm("norm_step", batch=16, tokens=8),
        # a training step over long sequences of an odd length, with all gradients
        _norm("norm_train", dtype="bf16", batch=4, tokens=4095, train=True, wide=True, case_seed=6),
        # a tree of 8 for one conversation: latency
        _attend("attend_single", batch=1, shortest=1900, longest=1900, nodes=8, page=16, share=1.0),
        # four drafted tokens of each request, long contexts: as many query rows as a small step has
        _attend("attend_few", dtype="fp16", batch=48, shortest=500, longest=12000, nodes=4, page=256, case_seed=7),
        # a tree of 16 for each request of a large batch with long contexts of very different lengths
        _attend("attend_batch"),
        # wide trees of an odd size over contiguous caches, narrow heads
        _attend("attend_wide", dtype="fp16", batch=12, shortest=300, longest=9000, nodes=61, heads=16, heads_kv=4, dim=64, page=0,
                case_seed=8),
        # one chain of drafts per conversation: latency
        _verify("verify_chain", batch=4, nodes=5, branch=0.0, vocabulary=32768),
        # trees for a large batch, an odd vocabulary, a draft model that is often wrong
        _verify("verify_trees", batch=64, nodes=24, vocabulary=100003, near=1.2, case_seed=9),
        # the caches of a small model and few conversations: latency
        _compact("compact_few", dtype="fp16", layers=4, batch=4, nodes=8, heads_kv=4, dim=64, case_seed=10),
        # all layers of a large batch
        _compact("compact_layers", layers=24, batch=96, nodes=32, page=64, case_seed=11),
        # a decoding step: what the rejected tokens took
        _release("release_step"),
        # a large offline batch, half of whose requests have ended
        _release("release_ended", requests=2048, longest=20000, whole=0.5, padding=999, case_seed=12),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("norm", "norm", "attend", "attend", "attend", "verify", "verify", "compact", "release"))
    c = None
    while c is None or _cost(c) > _LIMIT[kind]:
        dim, heads_kv = rng.choice((64, 128, 128, 256)), rng.choice((1, 2, 4, 8))
        heads = heads_kv * rng.choice((1, 2, 4, 8))
        seed, dtype = rng.randrange(1 << 20), rng.choice(("fp16", "bf16"))
        if kind == "norm":
            train = rng.random() < 0.5
            c = _norm("", dtype=rng.choice(("fp16", "bf16", "bf16", "fp32")), batch=_log_int(rng, 1, 64),
                      tokens=_log_int(rng, 64, 8192) if train else _log_int(rng, 1, 4096), heads=heads, heads_kv=heads_kv, dim=dim,
                      rotary=dim // rng.choice((1, 1, 2)), interleaved=rng.random() < 0.3, wide=rng.random() < 0.5, train=train,
                      case_seed=seed)
        elif kind == "attend":
            longest = _log_int(rng, 64, 32768)
            c = _attend("", dtype=dtype, batch=_log_int(rng, 1, 64), shortest=max(1, longest // rng.choice((1, 4, 32))), longest=longest,
                        nodes=_log_int(rng, 2, 128), share=rng.choice((0.5, 0.8, 1.0)), heads=heads, heads_kv=heads_kv, dim=dim,
                        page=rng.choice((0, 16, 32, 64, 128, 256)), case_seed=seed)
        elif kind == "verify":
            c = _verify("", dtype=rng.choice(("fp32", "fp32", "bf16", "fp16")), batch=_log_int(rng, 1, 64), nodes=_log_int(rng, 2, 64),
                        branch=rng.choice((0.0, 0.3, 0.6, 1.0)), vocabulary=_log_int(rng, 1000, 160000),
                        near=rng.choice((0.3, 0.7, 1.5)), case_seed=seed)
        elif kind == "compact":
            c = _compact("", dtype=dtype, layers=_log_int(rng, 1, 32), batch=_log_int(rng, 1, 96), cached=_log_int(rng, 16, 500),
                         nodes=_log_int(rng, 2, 64), heads_kv=heads_kv, dim=dim, page=rng.choice((0, 16, 24, 64, 256)), case_seed=seed)
        else:
            c = _release("", requests=_log_int(rng, 1, 2048), longest=_log_int(rng, 1, 20000), drafted=_log_int(rng, 1, 128),
                         whole=rng.choice((0.0, 0.1, 0.5)), page=rng.choice((16, 24, 32, 64, 256)),
                         padding=rng.choice((0, _log_int(rng, 1, 2000))), case_seed=seed)
    del c["name"]
    return c


# the most a drawn case of a kind may cost, in the units of _cost: that of its largest listed one
_LIMIT = {"norm": 4 * 4095 * 40 * 128 * 2.5, "attend": 32 * 16384 * 8 * 128 * 4 + 32 * 512 * 16384 * 4, "verify": 64 * 24 * 100003 * 8,
          "compact": 24 * 2 * 96 * 360 * 8 * 128, "release": 2048 * 20000 / 16}


def _cost(c):
    if c["kind"] == "norm":
        size = {"fp16": 1, "bf16": 1, "fp32": 2}[c["dtype"]] * (2.5 if c["train"] else 1)
        return size * c["batch"] * c["tokens"] * (c["heads"] + c["heads_kv"]) * c["dim"]
    if c["kind"] == "attend":
        return c["batch"] * c["longest"] * (c["heads_kv"] * c["dim"] * 4 + c["heads"] * c["nodes"] * 4)
    if c["kind"] == "verify":
        return c["batch"] * c["nodes"] * c["vocabulary"] * 8
    if c["kind"] == "compact":
        return c["layers"] * 2 * c["batch"] * (c["cached"] + c["nodes"] + c["page"] // 2) * c["heads_kv"] * c["dim"]
    return c["requests"] * c["longest"] / c["page"]


# ---- lengths and trees: numpy, from the case alone ----------------------------------------------------------------------------
def _rng(c):
    return np.random.default_rng(c["case_seed"])


def _trees(rng, batch, nodes, share, branch):
    """parents (batch, nodes): a request uses at least `share` of the nodes; `branch`: how often a node hangs below any earlier node
    instead of the one before it."""
    parents = np.full((batch, nodes), -1, dtype=np.int32)
    used = rng.integers(max(1, int(nodes * share)), nodes + 1, batch)
    for i in range(1, nodes):
        any_of = (rng.random(batch) * i).astype(np.int32)
        parents[:, i] = np.where(rng.random(batch) < branch, any_of, i - 1)
    parents[np.arange(nodes)[None, :] >= used[:, None]] = -1
    return parents


def _ancestors(parents):
    """seen (batch, nodes, nodes): node i sees j, itself or an ancestor; nodes that are not used see nothing."""
    batch, nodes = parents.shape
    seen = np.zeros((batch, nodes, nodes), dtype=bool)
    seen[:, 0, 0] = True
    at = np.arange(batch)
    for i in range(1, nodes):
        inside = parents[:, i] >= 0
        seen[:, i] = seen[at, np.maximum(parents[:, i], 0)] & inside[:, None]
        seen[:, i, i] = inside
    return seen


def _attend_plan(c):
    rng = _rng(c)
    lens = rng.integers(c["shortest"], c["longest"] + 1, c["batch"])
    return lens, _ancestors(_trees(rng, c["batch"], c["nodes"], c["share"], 0.5))


def _compact_plan(c):
    """(lengths, path (batch, nodes), accepted): the accepted nodes of each request, ascending, the root first."""
    rng = _rng(c)
    lens = rng.integers(1, c["cached"] + 1, c["batch"])
    accepted = rng.integers(1, c["nodes"] + 1, c["batch"])
    path = np.full((c["batch"], c["nodes"]), -1, dtype=np.int32)
    for b, n in enumerate(accepted):
        path[b, 0] = 0
        path[b, 1:n] = 1 + np.sort(rng.permutation(c["nodes"] - 1)[:n - 1])
    return lens, path, accepted


def _release_plan(c):
    """(tokens that pages are held for, tokens kept)."""
    rng = _rng(c)
    kept = rng.integers(1, c["longest"] + 1, c["requests"])
    held = kept + rng.integers(0, c["drafted"] + 1, c["requests"])
    kept[rng.random(c["requests"]) < c["whole"]] = 0
    return held, kept


def _pages(c, lens, page):
    """Block table of requests of these lengths from a shuffled pool with some pages to spare, and the pool's size.  A row ends in
    copies of its first page."""
    need = -(-lens // page)
    pool = int(need.sum()) + 8
    order = np.random.default_rng(c["case_seed"] + 1).permutation(pool).astype(np.int32)
    column = np.arange(int(need.max()))[None, :]
    first = np.cumsum(need) - need
    return order[first[:, None] + np.where(column < need[:, None], column, 0)], pool


# ---- inputs --------------------------------------------------------------------------------------------------------------------
def _values(gen, dtype, *shape):
    """Activations as projections give them: unit variance, a few channels much larger."""
    x = torch.randn(*shape, device="cuda", generator=gen)
    x *= 1 + 5 * (torch.rand(shape[-1], device="cuda", generator=gen) < 0.03)
    return x.to(dtype)


def _tables(longest, rotary, dtype):
    angle = torch.outer(torch.arange(longest, device="cuda", dtype=torch.float64),
                        10000.0 ** (-torch.arange(0, rotary, 2, device="cuda", dtype=torch.float64) / rotary))
    return angle.cos().to(dtype), angle.sin().to(dtype)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES.get(c.get("dtype"))
    s = dict(case=c)
    if c["kind"] == "norm":
        rng = _rng(c)
        B, T, D = c["batch"], c["tokens"], c["dim"]
        s["q"], s["k"] = _values(gen, dt, B, T, c["heads"], D), _values(gen, dt, B, T, c["heads_kv"], D)
        table = torch.float32 if c["wide"] else dt
        s["q_weight"], s["k_weight"] = ((1 + 0.3 * torch.randn(D, device="cuda", generator=gen)).to(table) for _ in range(2))
        s["cos"], s["sin"] = _tables(c["longest"], c["rotary"], table)
        if c["train"]:
            s["positions"] = None                       # those of the sequence
            s["dq"], s["dk"] = _values(gen, dt, B, T, c["heads"], D), _values(gen, dt, B, T, c["heads_kv"], D)
            for name in ("q", "k", "q_weight", "k_weight"):
                s[name].requires_grad_()
        else:                                           # each token at its depth behind the context
            first = rng.integers(0, c["longest"] - T, B)
            depth = np.minimum(rng.integers(0, T, (B, T)), np.arange(T)[None, :])
            s["positions"] = torch.from_numpy((first[:, None] + depth).astype(np.int32)).cuda()
        return s
    if c["kind"] == "verify":
        B, N, V = c["batch"], c["nodes"], c["vocabulary"]
        parents = _trees(_rng(c), B, N, 0.7, c["branch"])
        draft = torch.empty(B, N, V, dtype=dt, device="cuda")
        target = torch.empty_like(draft)
        tokens = torch.zeros(B, N, dtype=torch.int64, device="cuda")
        above = torch.from_numpy(np.maximum(parents, 0)).cuda().long()
        for b in range(B):
            logits = 4 * torch.randn(N, V, device="cuda", generator=gen)
            q = torch.softmax(logits, -1)
            logits += c["near"] * torch.randn(N, V, device="cuda", generator=gen)
            draft[b], target[b] = q, torch.softmax(logits, -1)
            # a node's token is drawn from the distribution at its parent
            drawn = torch.rand(N, 1, device="cuda", generator=gen)
            sums = torch.cumsum(q, -1)
            tokens[b] = torch.searchsorted(sums[above[b]], drawn * sums[above[b], -1:], right=True).clamp_(max=V - 1)[:, 0]
        s.update(tokens=tokens, parents=torch.from_numpy(parents).cuda(), target=target, draft=draft,
                 accept=torch.rand(B, N, device="cuda", generator=gen), sample=torch.rand(B, device="cuda", generator=gen))
        return s
    if c["kind"] == "release":
        held, kept = _release_plan(c)
        table, pool = _pages(c, held, c["page"])
        table = torch.randperm(pool, device="cuda", generator=gen).to(torch.int32)[torch.from_numpy(table).cuda().long()]
        freed = int((-(-held // c["page"]) - -(-kept // c["page"])).sum())
        s.update(held=torch.tensor(held, dtype=torch.int32, device="cuda"), kept=torch.tensor(kept, dtype=torch.int32, device="cuda"),
                 table=table, room=freed + c["padding"])
        return s
    plan = _attend_plan(c) if c["kind"] == "attend" else _compact_plan(c)
    lens, N = plan[0], c["nodes"]
    s["cache_seqlens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if c["page"]:
        table, pool = _pages(c, lens + N, c["page"])
        s["table"], shape = torch.from_numpy(table).cuda(), (pool, c["page"], c["heads_kv"], c["dim"])
    else:
        s["table"], shape = None, (c["batch"], int(lens.max()) + N, c["heads_kv"], c["dim"])
    if c["kind"] == "compact":
        s["caches"] = [[torch.randn(shape, device="cuda", dtype=dt, generator=gen) for _ in range(c["layers"])] for _ in range(2)]
        s["path"] = torch.from_numpy(plan[1]).cuda()
        s["accepted"] = torch.tensor(plan[2], dtype=torch.int32, device="cuda")
        return s
    s["k_cache"], s["v_cache"] = (torch.randn(shape, device="cuda", dtype=dt, generator=gen) for _ in range(2))
    s["q"] = _values(gen, dt, c["batch"], N, c["heads"], c["dim"])
    s["k"], s["v"] = (_values(gen, dt, c["batch"], N, c["heads_kv"], c["dim"]) for _ in range(2))
    s["mask"] = torch.from_numpy(plan[1]).cuda()
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------------------
def _halves(x, rotary, interleaved):
    return (x[..., 0:rotary:2], x[..., 1:rotary:2]) if interleaved else (x[..., :rotary // 2], x[..., rotary // 2:rotary])


def _rotate(x, cos, sin, interleaved):
    """x (batch, tokens, heads, dim), cos and sin (batch or 1, tokens, 1, rotary / 2)."""
    rotary = 2 * cos.shape[-1]
    a, b = _halves(x, rotary, interleaved)
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., rotary:]), -1)


_EPS = 1e-6


def _plain_norm(x, weight, cos, sin, interleaved, grad):
    """The output of one of q and k, and with `grad` the gradients of x and weight."""
    wide, w = x.float(), weight.float()
    inverse = torch.rsqrt((wide * wide).mean(-1, keepdim=True) + _EPS)
    unit = wide * inverse
    out = _rotate(unit * w, cos, sin, interleaved).to(x.dtype)
    if grad is None:
        return out, None, None
    dy = _rotate(grad.float(), cos, -sin, interleaved)
    dweight = (dy * unit).sum((0, 1, 2))
    dy *= w
    dx = inverse * (dy - unit * (dy * unit).mean(-1, keepdim=True))
    return out, dx.to(x.dtype), dweight.to(weight.dtype)


def _rows_of(positions, seq, table, shape, page):
    """Flat rows of a cache for these positions of requests `seq`."""
    if table is None:
        return seq * shape[1] + positions
    return table[seq, positions // page].long() * page + positions % page


def _plain_attend(q, k_cache, v_cache, table, lens, mask):
    """q (batch, nodes, heads, dim): the last tokens of sequences of `lens` tokens behind them."""
    batch, nodes, heads, dim = q.shape
    heads_kv = k_cache.shape[2]
    if table is None:
        k, v = k_cache.float(), v_cache.float()
    else:
        k, v = (x[table].flatten(1, 2).float() for x in (k_cache, v_cache))
    q = q.float().view(batch, nodes, heads_kv, heads // heads_kv, dim)
    scores = torch.einsum("bthgd,bkhd->bhgtk", q, k) / math.sqrt(dim)
    del k
    node = torch.arange(scores.shape[-1], device=q.device)[None, :] - lens[:, None]         # of a key; context below 0
    inside = ((node >= 0) & (node < nodes))[:, None, :]
    seen = torch.gather(mask, 2, node.clamp(0, nodes - 1)[:, None, :].expand(-1, nodes, -1)) & inside
    seen |= (node < 0)[:, None, :]
    scores.masked_fill_(~seen[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = scores.sum(-1).permute(0, 3, 1, 2)[..., None]
    out = torch.einsum("bhgtk,bkhd->bthgd", scores, v)
    return torch.where(total > 0, out / total, 0.0).reshape(batch, nodes, heads, dim)


def _plain_verify(tokens, parents, target, draft, accept, sample):
    batch, nodes, size = target.shape
    at = torch.arange(batch, device=target.device)
    node = torch.zeros(batch, dtype=torch.int64, device=target.device)
    count = torch.ones_like(node)
    path = torch.full((batch, nodes + 1), -1, dtype=torch.int32, device=target.device)
    path[:, 0] = 0
    # what is left of the target's distribution at `node` is max(p - less q, 0), of mass `mass`
    less = torch.zeros(batch, dtype=torch.float64, device=target.device)
    mass = torch.ones_like(less)
    rest = None
    for i in range(1, nodes):
        child = parents[:, i] == node
        token = tokens[:, i]
        p, q = target[at, node, token].double(), draft[at, node, token].double()
        taken = child & (accept[:, i].double() * q * mass < (p - less * q).clamp_min(0))
        lost = child & ~taken
        less = torch.where(lost, less + mass, less)
        rest = (target[at, node].double() - less[:, None] * draft[at, node].double()).clamp_min_(0)
        mass = torch.where(lost, rest.sum(-1), mass)
        path[at, torch.where(taken, count, nodes)] = i
        node, count = torch.where(taken, i, node), count + taken
        less, mass = torch.where(taken, 0.0, less), torch.where(taken, 1.0, mass)
    p = target[at, node].double()
    rest = (p - less[:, None] * draft[at, node].double()).clamp_min_(0)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, p)
    sums = torch.cumsum(rest, -1)
    token = (sums <= sample.double()[:, None] * sums[:, -1:]).sum(-1)
    last = torch.where(rest > 0, torch.arange(size, device=p.device), -1).amax(-1)
    return path[:, :nodes], count.to(torch.int32), torch.minimum(token, last)


def _plain_release(held, kept, table, page, room):
    first, end = (kept + page - 1) // page, (held + page - 1) // page
    column = torch.arange(table.shape[1], device=table.device)[None, :]
    given = (column >= first[:, None]) & (column < end[:, None])
    where = torch.cumsum(given.flatten(), 0).view_as(given) - 1
    pages = torch.full((room + 1,), -1, dtype=torch.int32, device=table.device)
    pages[torch.where(given, where, room)] = table
    pages[room] = -1
    return pages[:room], given.sum(dtype=torch.int32)


def run(state):
    s, c = state, state["case"]
    if own:
        import flash_attn_triton_b200 as fa
    if c["kind"] == "norm":
        if own:
            out = fa.qk_norm_rotary(s["q"], s["k"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], positions=s["positions"], eps=_EPS,
                                    rotary_interleaved=c["interleaved"])
            if not c["train"]:
                return out
            return (*out, *torch.autograd.grad(out, (s["q"], s["k"], s["q_weight"], s["k_weight"]), (s["dq"], s["dk"])))
        at = slice(0, c["tokens"]) if c["train"] else s["positions"].long()
        with torch.no_grad():
            cos, sin = (x[at].float().view(-1, c["tokens"], 1, c["rotary"] // 2) for x in (s["cos"], s["sin"]))
            q, dq, dqw = _plain_norm(s["q"], s["q_weight"], cos, sin, c["interleaved"], s.get("dq"))
            k, dk, dkw = _plain_norm(s["k"], s["k_weight"], cos, sin, c["interleaved"], s.get("dk"))
        return (q, k, dq, dk, dqw, dkw) if c["train"] else (q, k)
    if c["kind"] == "verify":
        given = s["tokens"], s["parents"], s["target"], s["draft"], s["accept"], s["sample"]
        return fa.verify_draft_tree(*given) if own else _plain_verify(*given)
    if c["kind"] == "release":
        given = s["held"], s["kept"], s["table"], c["page"], s["room"]
        return fa.release_pages(*given) if own else _plain_release(*given)
    lens, table = s["cache_seqlens"], s["table"]
    if c["kind"] == "compact":
        if own:
            fa.kvcache_compact(*s["caches"], lens, s["path"], s["accepted"], block_table=table)
            return s["caches"]
        seq = torch.arange(c["batch"], device=lens.device)[:, None].expand(-1, c["nodes"])
        step = torch.arange(c["nodes"], device=lens.device)[None, :]
        source = torch.where(step < s["accepted"][:, None], s["path"], step).long()         # the others stay where they are
        for x in (x for one in s["caches"] for x in one):
            rows = x.view(-1, c["heads_kv"] * c["dim"])
            rows[_rows_of(lens[:, None] + step, seq, table, x.shape, c["page"])] = \
                rows[_rows_of(lens[:, None] + source, seq, table, x.shape, c["page"])]
        return s["caches"]
    caches = s["k_cache"], s["v_cache"]
    if own:
        out = fa.flash_attn_with_kvcache(s["q"], *caches, s["k"], s["v"], cache_seqlens=lens, block_table=table, tree_mask=s["mask"])
        return (out, *caches)
    seq = torch.arange(c["batch"], device=lens.device)[:, None]
    rows = _rows_of(lens[:, None] + torch.arange(c["nodes"], device=lens.device), seq, table, caches[0].shape, c["page"])
    for cache, x in zip(caches, (s["k"], s["v"])):
        cache.view(-1, c["heads_kv"], c["dim"])[rows] = x
    return (_plain_attend(s["q"], *caches, table, lens, s["mask"]).to(s["q"].dtype), *caches)


def work(case):
    """Bytes: what is read, once, and what is written, once.  Operations: two products per visible pair of an attention, a few per
    element of the others."""
    c = case
    size = {"fp16": 2, "bf16": 2, "fp32": 4}.get(c.get("dtype"))
    if c["kind"] == "norm":
        tokens = c["batch"] * c["tokens"]
        elements, table = tokens * (c["heads"] + c["heads_kv"]) * c["dim"], 4 if c["wide"] else size
        rows = 2.0 * table * c["rotary"] / 2 * min(c["tokens"] if c["train"] else tokens, c["longest"])
        if not c["train"]:
            return {"bytes": 2.0 * elements * size + rows + 4.0 * tokens, "flops": 7.0 * elements}
        # forward and backward: both read x, and the tables
        return {"bytes": 5.0 * elements * size + 2 * rows, "flops": 25.0 * elements}
    if c["kind"] == "verify":
        # both distributions at the node where the path of a request ends
        return {"bytes": 2.0 * c["batch"] * c["vocabulary"] * size + 20.0 * c["batch"] * c["nodes"],
                "flops": 4.0 * c["batch"] * c["vocabulary"]}
    if c["kind"] == "release":
        held, kept = _release_plan(c)
        freed = int((-(-held // c["page"]) - -(-kept // c["page"])).sum())
        return {"bytes": 8.0 * c["requests"] + 4.0 * (2 * freed + c["padding"]) + 4, "flops": 4.0 * (freed + c["requests"])}
    row = c["heads_kv"] * c["dim"] * size
    if c["kind"] == "compact":
        _, path, accepted = _compact_plan(c)
        step = np.arange(c["nodes"])[None, :]
        moved = int(((step < accepted[:, None]) & (path != step)).sum())
        return {"bytes": 2.0 * 2 * c["layers"] * moved * row + 4.0 * int(accepted.sum()) + 8.0 * c["batch"], "flops": 0.0}
    lens, seen = _attend_plan(c)
    tokens = c["batch"] * c["nodes"]
    cache = 2.0 * int(lens.sum()) * row
    new = 2 * 2.0 * tokens * row
    q = 2.0 * tokens * c["heads"] * c["dim"] * size
    pairs = int(lens.sum()) * c["nodes"] + int(seen.sum())
    return {"bytes": cache + new + q + tokens * c["nodes"], "flops": 4.0 * c["dim"] * c["heads"] * pairs}


# ---- the same in 64 bits ---------------------------------------------------------------------------------------------------
def _exact_turn(c, x, weight, cos, sin):
    """The definition, pair by pair as complex numbers."""
    y = x / (x.square().sum(-1, keepdim=True) / c["dim"] + _EPS).sqrt() * weight
    r = c["rotary"]
    first, second = (y[..., :r:2], y[..., 1:r:2]) if c["interleaved"] else y[..., :r].chunk(2, -1)
    turned = torch.complex(first, second) * torch.complex(cos, sin)[:, :, None]
    parts = (turned.real, turned.imag)
    turned = torch.stack(parts, -1).flatten(-2) if c["interleaved"] else torch.cat(parts, -1)
    return torch.cat((turned, y[..., r:]), -1)


def exact(case, seed):
    """Norms, rotations and attention from their definitions in 64 bits; whole numbers and moved rows have none."""
    c = case
    if c["kind"] not in ("norm", "attend"):
        return None
    s = prepare(case, seed)
    if c["kind"] == "norm":
        place = s["positions"] if s["positions"] is not None else torch.arange(c["tokens"], device="cuda")[None].expand(c["batch"], -1)
        cos, sin = s["cos"].double()[place.long()], s["sin"].double()[place.long()]
        outs, grads = [], []
        for x, w, g in (("q", "q_weight", "dq"), ("k", "k_weight", "dk")):
            leaves = [s[n].detach().double().requires_grad_(c["train"]) for n in (x, w)]
            out = _exact_turn(c, *leaves, cos, sin)
            outs.append(out.detach())
            if c["train"]:
                grads.append(torch.autograd.grad(out, leaves, s[g].double()))
        return (*outs, grads[0][0], grads[1][0], grads[0][1], grads[1][1]) if c["train"] else tuple(outs)
    lens, seen = _attend_plan(c)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group, N = c["heads"] // c["heads_kv"], c["nodes"]
    for b, n in enumerate(lens.tolist()):
        place = torch.arange(n, device="cuda")
        if s["table"] is None:
            page, row = torch.full_like(place, b), place
        else:
            page, row = s["table"][b].long()[place // c["page"]], place % c["page"]
        hidden = ~torch.from_numpy(seen[b]).cuda()
        for h in range(c["heads_kv"]):
            k = torch.cat((s["k_cache"][page, row, h], s["k"][b, :, h])).double()
            v = torch.cat((s["v_cache"][page, row, h], s["v"][b, :, h])).double()
            heads = slice(h * group, (h + 1) * group)
            logits = s["q"][b, :, heads].double() @ k.T * c["dim"] ** -0.5
            logits[..., n:].masked_fill_(hidden[:, None, :], -math.inf)
            out[b, :, heads] = torch.softmax(logits, -1) @ v
    # rows of the cache are copies
    return out, None, None
