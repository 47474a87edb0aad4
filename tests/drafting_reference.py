"""Decoding with drafted trees in 64 bits, from the definitions: CPU tensors in, CPU tensors out."""
import math

import torch


def turn(x, cos, sin, interleaved):
    """x (..., tokens, heads, dim), cos and sin (..., tokens, rotary / 2): the pairs rotated, and the magnitude that was added up."""
    r = 2 * cos.shape[-1]
    cos, sin = cos[..., None, :], sin[..., None, :]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    parts = a * cos - b * sin, a * sin + b * cos
    sizes = (a * cos).abs() + (b * sin).abs(), (a * sin).abs() + (b * cos).abs()

    def joined(two, rest):
        two = torch.stack(two, -1).flatten(-2) if interleaved else torch.cat(two, -1)
        return torch.cat((two, rest), -1)
    return joined(parts, x[..., r:]), joined(sizes, x[..., r:].abs())


def norm(x, weight, cos, sin, interleaved, eps, grad=None):
    """(out, size of out), and with grad also (dx, size of dx, dweight, size of dweight); in doubles."""
    unit = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    out, size = turn(unit * weight, cos, sin, interleaved)
    if grad is None:
        return out, size
    g, g_size = turn(grad, cos, -sin, interleaved)
    h, h_size = g * weight, g_size * weight.abs()
    inverse = 1 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    dx = inverse * (h - unit * (h * unit).mean(-1, keepdim=True))
    dx_size = inverse * (h_size + unit.abs() * (h_size * unit.abs()).mean(-1, keepdim=True))
    dims = tuple(range(x.ndim - 1))
    return out, size, dx, dx_size, (g * unit).sum(dims), (g_size * unit.abs()).sum(dims)


def attend(q, k, v, seen, scale):
    """q (rows, heads, dim), k and v (keys, heads_kv, dim), seen (rows, keys): out and the sum of the magnitudes, rows that see
    nothing are 0.  Keys that a row does not see are no part of its sums."""
    rows, heads, dim = q.shape
    group = heads // k.shape[1]
    out, size = torch.zeros(rows, heads, dim, dtype=torch.float64), torch.zeros(rows, heads, dim, dtype=torch.float64)
    for i in range(rows):
        at = torch.nonzero(seen[i])[:, 0]
        if len(at) == 0:
            continue
        for h in range(heads):
            p = torch.softmax(k[at, h // group].double() @ q[i, h].double() * scale, 0)
            vals = v[at, h // group].double()
            out[i, h], size[i, h] = p @ vals, p @ vals.abs()
    return out, size


def verify(tokens, parents, target, draft, accept, sample):
    """One request: (path, next token), the distributions normalised after every rejection."""
    target, draft, accept = target.double(), draft.double(), accept.double()
    vocab = target.shape[1]
    path, p, fresh = [0], target[0].clamp_min(0), True
    for i in range(1, len(parents)):
        if int(parents[i]) != path[-1]:
            continue
        x, q = int(tokens[i]), draft[path[-1]]
        px, qx = (float(p[x]), float(q[x])) if 0 <= x < vocab else (0.0, 0.0)
        if float(accept[i]) * qx < px:
            path.append(i)
            p, fresh = target[i].clamp_min(0), True
            continue
        rest = (p - q).clamp_min(0)
        total = rest.sum()
        p = rest / total if total > 0 else rest
        fresh = False
    if not fresh and float(p.sum()) == 0.0:
        p = target[path[-1]].clamp_min(0)
    total = p.sum()
    if not (total > 0) or math.isinf(float(total)):
        return path, -1
    sums = torch.cumsum(p, 0)
    over = torch.nonzero(sums > float(sample) * total)
    return path, int(over[0, 0]) if len(over) else int(torch.nonzero(p > 0)[-1, 0])


def tree(gen, batch, nodes, used=None, branch=0.5):
    """(parents, seen): nodes from `used` on are not part of the tree and see nothing."""
    parents = torch.full((batch, nodes), -1, dtype=torch.int32)
    seen = torch.zeros(batch, nodes, nodes, dtype=torch.bool)
    for b in range(batch):
        n = nodes if used is None else used[b]
        for i in range(n):
            seen[b, i, i] = True
            if i:
                up = int(torch.randint(i, (1,), generator=gen)) if float(torch.rand(1, generator=gen)) < branch else i - 1
                parents[b, i] = up
                seen[b, i] |= seen[b, up]
    return parents, seen
