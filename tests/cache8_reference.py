"""The 8-bit KV cache in plain form on the CPU: append by the exact fp32 rule, attention in 64 bits."""
import math

import torch

LARGEST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
TINY = torch.finfo(torch.float32).tiny


def bits(codes):
    """Codes as bytes: NaN patterns compare too."""
    return codes.view(torch.int8)


def coded(x, dtype):
    """fp32 -> nearest code."""
    x = x.clamp(-LARGEST[dtype], LARGEST[dtype])
    return x.round().to(torch.int8) if dtype == torch.int8 else x.to(dtype)


def append_run(x, cache, scale, page, row, kept=None):
    """Tokens x (n, heads, d) to rows row, row + 1, ... of a page, all of them in one block; `kept` rows before them stay (all, if None)."""
    rows = cache.shape[1] // scale.shape[1]
    block, at = row // rows, row % rows
    assert at + len(x) <= rows
    kept = at if kept is None else kept
    x = x.float()
    old = scale[page, block].clone() if kept else torch.zeros(x.shape[1])
    need = x.abs().amax(dim=(0, 2)) / torch.tensor(LARGEST[cache.dtype])
    need = torch.where(need < TINY, torch.zeros(()), need)
    now = torch.maximum(old, need)
    inv = torch.where(now > 0, 1 / now, torch.zeros(()))
    for h in range(x.shape[1]):
        if kept and now[h] > old[h]:
            held = cache[page, row - kept:row, h].float() * (old[h] * inv[h])
            cache[page, row - kept:row, h] = coded(held, cache.dtype)
        cache[page, row:row + len(x), h] = coded(x[:, h] * inv[h], cache.dtype)
    scale[page, block] = now


def append_slots(x, cache, scale, slots):
    """Packed tokens by slot; runs of one block."""
    rows, size = cache.shape[1] // scale.shape[1], cache.shape[1]
    slots = slots.tolist()
    i = 0
    while i < len(slots):
        if slots[i] < 0:
            i += 1
            continue
        j = i + 1
        while j < len(slots) and slots[j] == slots[j - 1] + 1 and slots[j] % rows:
            j += 1
        append_run(x[i:j], cache, scale, slots[i] // size, slots[i] % size)
        i = j


def append_call(x, cache, scale, old, table=None, batch_idx=None, leftpad=None):
    """The new tokens x (batch, n, heads, d) of a cache call behind `old` tokens of each sequence."""
    rows, size = cache.shape[1] // scale.shape[1], cache.shape[1]
    for b in range(x.shape[0]):
        pad = 0 if leftpad is None else int(leftpad[b])
        i, n = 0, x.shape[1]
        while i < n:
            pos = int(old[b]) + i + pad
            page = int(table[b, pos // size]) if table is not None else b if batch_idx is None else int(batch_idx[b])
            row = pos % size if table is not None else pos
            m = min(rows - row % rows, n - i)
            append_run(x[b, i:i + m], cache, scale, page, row, min(row % rows, int(old[b]) + i))
            i += m


def values(cache, scale):
    """What the cache holds, in 64 bits."""
    return cache.double() * scale.double().repeat_interleave(cache.shape[1] // scale.shape[1], dim=1)[..., None]


def gathered(x, length, b, table=None, batch_idx=None, leftpad=None):
    if table is not None:
        return x[table[b].long()].flatten(0, 1)[:length]
    pad = 0 if leftpad is None else int(leftpad[b])
    return x[b if batch_idx is None else int(batch_idx[b]), pad:pad + length]


def attend(q, k_values, v_values, lengths, softmax_scale=None, causal=False, window=(-1, -1), alibi=None, **place):
    """(out, sum_j p_j |v_j|) in 64 bits; q the last tokens of sequences of `lengths` tokens.  Rows that see nothing are 0."""
    B, n, H, D = q.shape
    out, weight = torch.zeros(B, n, H, D, dtype=torch.float64), torch.zeros(B, n, H, D, dtype=torch.float64)
    group = H // k_values.shape[2]
    for b in range(B):
        length = int(lengths[b])
        k, v = gathered(k_values, length, b, **place), gathered(v_values, length, b, **place)
        at = torch.arange(length - n, length)[:, None]
        key = torch.arange(length)[None, :]
        hidden = torch.zeros(n, length, dtype=torch.bool)
        if causal:
            hidden |= key > at
        if window[0] >= 0:
            hidden |= key < at - window[0]
        if window[1] >= 0:
            hidden |= key > at + window[1]
        empty = hidden.all(-1) if length else torch.ones(n, dtype=torch.bool)
        for h in range(H):
            s = (q[b, :, h].double() @ k[:, h // group].T) * (D ** -0.5 if softmax_scale is None else softmax_scale)
            if alibi is not None:
                s = s - float(alibi[b, h]) * (at - key).abs()
            # (columns are taken one by one where a value is hidden from some rows: 0 times infinity)
            s = s.masked_fill(hidden, -math.inf)
            p = torch.softmax(s, -1).masked_fill(hidden, 0.0)
            vh = v[:, h // group]
            if torch.isfinite(vh).all():
                out[b, :, h], weight[b, :, h] = p @ vh, p @ vh.abs()
            else:
                for i in range(n):
                    seen = ~hidden[i]
                    out[b, i, h], weight[b, i, h] = p[i, seen] @ vh[seen], p[i, seen] @ vh[seen].abs()
            out[b, empty, h] = weight[b, empty, h] = 0.0
    return out, weight


def tolerance(out, weight, dtype, keys, largest):
    """Weights are rounded to fp16 once (half a step is 2^-11 of a weight, and 2^-25 of the largest where they are tiny); exponents and
    sums in fp32 are off by less than 2^-15 of a weight for scores up to 60; the result is rounded once to its type."""
    return (2.0 ** -11 + 2.0 ** -15) * weight + keys * 2.0 ** -25 * largest + torch.finfo(dtype).eps / 2 * out.abs() + 1e-12
