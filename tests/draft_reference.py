"""Trees of drafts in 64 bits, from their definitions: what the kernels are compared with."""

import numpy as np
import torch

import paged_reference as R


def parent_of(i, parents):
    """The node that node i hangs on, or -1."""
    a = int(parents[i])
    return a if 0 <= a < i else -1


def tree(parents, most):
    """(seen [n, n] bool, depth [n]) of one request; nodes from `most` on see none of the tree."""
    n = len(parents)
    seen, depth = torch.zeros(n, n, dtype=torch.bool), [0] * n
    for i in range(min(n, most)):
        a = parent_of(i, parents)
        if a >= 0:
            seen[i], depth[i] = seen[a], depth[a] + 1
        seen[i, i] = True
    return seen, depth


def words(seen, count):
    """Rows of bits as lists of `count` signed 64-bit words."""
    out = []
    for row in seen.tolist():
        w = [sum(1 << (j % 64) for j, x in enumerate(row) if x and j // 64 == i) for i in range(count)]
        out.append([x - (1 << 64) if x >> 63 else x for x in w])
    return out


def mass(x):
    """Probabilities as they count."""
    x = np.asarray(x, np.float64)
    return np.where(np.isfinite(x) & (x > 0), x, 0.0)


def verify(p, tokens, parents, u, q=None):
    """One request: (path, next token).  p and q [n, V] in 64 bits, u [n]."""
    n = len(tokens)
    if n == 0:
        return [], -1
    path, v = [0], p.shape[1]
    while True:
        x = path[-1]
        rest, m, after = mass(p[x]), 1.0, None
        for c in range(x + 1, min(n, 1024)):
            if parent_of(c, parents) != x:
                continue
            known = 0 <= tokens[c] < v
            r = rest[tokens[c]] if known else 0.0
            if q is None:
                if u[c] * m < r:
                    after = c
                    break
                m = max(m - r, 0.0)
                if known:
                    rest = rest.copy()
                    rest[tokens[c]] = 0.0
            else:
                row = mass(q[x])
                if u[c] * (row[tokens[c]] if known else 0.0) * m < r:
                    after = c
                    break
                rest = np.maximum(rest / m - row, 0.0) if m > 0 else np.zeros(v)
                m = rest.sum()
        if after is None:
            break
        path.append(after)
    if not rest.sum() > 0:
        rest = mass(p[path[-1]])
    above = np.flatnonzero(np.cumsum(rest) > u[0] * rest.sum())
    some = np.flatnonzero(rest > 0)
    return path, int(above[0]) if len(above) else int(some[-1]) if len(some) else 0


def keep_path(path, n, length, row, codes, scale, block):
    """Move one request's path in one layer: codes [blocks, Hk, block, D] as values and scale [blocks, Hk] in 64 bits, in place.
    Returns the tokens to keep."""
    base = length - n
    good = 0
    while good < len(path) and (path[good - 1] if good else -1) < path[good] < n:
        good += 1
    path = path[:good]
    if base >= 0:
        into = {}
        for j, a in enumerate(path):
            if a != j:
                into.setdefault((base + j) // block, []).append(((base + j) % block, base + a))
        at = lambda e: int(row[e]) if e < len(row) and 0 <= int(row[e]) < codes.shape[0] else -1
        for e in sorted(into):
            b = at(e)
            if b < 0:
                continue
            moves = [(o, at(src // block), src % block) for o, src in into[e]]
            first, was = moves[0][0], scale[b].clone()
            moves = [(o, codes[sb, :, so].clone(), scale[sb].clone()) for o, sb, so in moves if sb >= 0]
            now = was.clone()
            for o, x, s in moves:
                v = (x * s[:, None]).abs()
                v = torch.where(torch.isfinite(v), v, torch.zeros_like(v)).amax(1)
                now = torch.where((s > was) & (v > 0), torch.maximum(now, R.scale_of(v)), now)
            grown = now != was
            if bool(grown.any()):
                codes[b, grown, :first] = R.nearest_e4m3(codes[b, grown, :first] * (was[grown] / now[grown])[:, None, None])
            for o, x, s in moves:
                codes[b, :, o] = torch.where(((s == now) | (now == 0))[:, None], x, R.nearest_e4m3(x * (s / now)[:, None]))
            scale[b] = now
    return max(base + len(path), 0)


def turn(x, cos, sin):
    """Half-split rotation of x [..., D] by cos and sin [..., D/2]."""
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def turned_size(x, cos, sin):
    """What a rotation, either way, adds up at most."""
    a, b = x.abs().chunk(2, -1)
    return torch.cat([a * cos.abs() + b * sin.abs(), b * cos.abs() + a * sin.abs()], -1)


def norm_rope(x, w, cos, sin, eps):
    """x [..., D] in 64 bits: (result, x r, r)."""
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return turn(x * r * w, cos, sin), x * r, r


def norm_rope_grads(x, w, cos, sin, eps, g):
    """(gradient of x, gradient of w [D], g turned back, x r, r)."""
    _, n, r = norm_rope(x, w, cos, sin, eps)
    g = turn(g, cos, -sin)
    gw = g * w
    mean = (gw * n).mean(-1, keepdim=True)
    return r * (gw - n * mean), (g * n).flatten(0, -2).sum(0), g, n, r
