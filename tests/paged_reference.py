"""The paged 8-bit cache in 64 bits, token by token: what its kernels are compared with."""

import math

import torch

LOW = -110


def scale_of(amax):
    """Smallest power of two 2^e, e >= -110, with amax <= 448 * 2^e (fp64 in and out)."""
    out = torch.empty_like(amax)
    for i, a in enumerate(amax.flatten().tolist()):
        e = LOW
        if a > 0:
            f, x = math.frexp(a)
            e = max(LOW, x - 9 if f <= 0.875 else x - 8)
        out.view(-1)[i] = 2.0 ** e
    return out


def nearest_e4m3(x):
    """Nearest e4m3 value, ties to even, saturating; NaN stays (fp64 in and out)."""
    _, e = torch.frexp(x.abs().clamp(2.0 ** -6, 448.0))
    step = torch.exp2((e - 4).to(x.dtype))
    return (torch.round(x.clamp(-448, 448) / step) * step).clamp(-448, 448)


def blocks_of(n, block):
    return -(-n // block)


def reserve(new, st, slots, block):
    """``paged_kv_reserve`` on a dict of lengths, table, free, count; returns (slot_map, positions, cu, shortage)."""
    n = [max(0, int(x)) for x in new]
    held = [int(x) for x in st["lengths"]]
    need = [blocks_of(h + a, block) - blocks_of(h, block) for h, a in zip(held, n)]
    slot_map, pos = [-1] * slots if slots < 10 ** 6 else None, [0] * (slots if slots < 10 ** 6 else 0)
    width = st["table"].shape[1]
    if sum(need) > st["count"] or sum(n) > slots or any(blocks_of(h + a, block) > width for h, a in zip(held, n)):
        return slot_map, pos, [0] * (len(n) + 1), 1
    cu, t = [0], 0
    for r, a in enumerate(n):
        for j in range(blocks_of(held[r], block), blocks_of(held[r] + a, block)):
            st["count"] -= 1
            st["table"][r, j] = st["free"][st["count"]]
        for p in range(held[r], held[r] + a):
            if slot_map is not None:
                slot_map[t], pos[t] = int(st["table"][r, p // block]) * block + p % block, p
            t += 1
        st["lengths"][r] = held[r] + a
        cu.append(t)
    return slot_map, pos, cu, 0


def trim(keep, st, block):
    """``paged_kv_trim`` on the same dict."""
    gone = []
    for r, k in enumerate(keep):
        held = int(st["lengths"][r])
        k = min(max(0, int(k)), held)
        for j in range(blocks_of(k, block), blocks_of(held, block)):
            gone.append(int(st["table"][r, j]))
            st["table"][r, j] = -1
        st["lengths"][r] = k
    for b in reversed(gone):
        st["free"][st["count"]] = b
        st["count"] += 1


def write(x, slots, codes, scale, block):
    """``fp8_kv_write`` of one operand: x [T, Hk, D] fp64, codes [blocks, Hk, block, D] as values and scale [blocks, Hk], in place."""
    slots, t = [int(s) for s in slots], 0
    inside = lambda s: 0 <= s < codes.shape[0] * block
    while t < len(slots):
        if not inside(slots[t]):
            t += 1
            continue
        e = t + 1
        while e < len(slots) and slots[e] == slots[e - 1] + 1 and slots[e] % block != 0 and inside(slots[e]):
            e += 1
        b, at = slots[t] // block, slots[t] % block
        part = x[t:e].transpose(0, 1)
        size = torch.where(torch.isfinite(part), part.abs(), torch.zeros_like(part))
        now = scale_of(size.amax(dim=(1, 2)))
        if at > 0:
            now = torch.maximum(now, scale[b])
            codes[b, :, :at] = nearest_e4m3(codes[b, :, :at] * (scale[b] / now)[:, None, None])
        codes[b, :, at:at + e - t] = nearest_e4m3(part / now[:, None, None])
        scale[b] = now
        t = e


def attend(q, k, v, limits, scaling, g):
    """q [n, H, D], k and v [Hk, S, D] fp64; token i sees the first limits[i] keys.  (out [n, H, D], lse [n, H])"""
    n, h, d = q.shape
    out, lse = torch.zeros_like(q), torch.full((n, h), -math.inf, dtype=q.dtype)
    for i in range(n):
        seen = max(0, min(int(limits[i]), k.shape[1]))
        if seen == 0:
            continue
        kk = k[:, :seen].repeat_interleave(g, 0)
        vv = v[:, :seen].repeat_interleave(g, 0)
        s = torch.einsum("hd,hsd->hs", q[i], kk) * scaling
        lse[i] = torch.logsumexp(s, 1)
        out[i] = torch.einsum("hs,hsd->hd", torch.exp(s - lse[i][:, None]), vv)
    return out, lse


def gather(codes, scale, row, length, block):
    """Values [Hk, length, D] of one request's keys or values."""
    ids = [int(row[j]) for j in range(blocks_of(length, block))]
    if not ids:
        return torch.zeros(codes.shape[1], 0, codes.shape[3], dtype=torch.float64)
    x = codes[ids].double() * scale[ids].double()[:, :, None, None]
    return x.transpose(0, 1).flatten(1, 2)[:, :length]
