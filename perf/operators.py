"""Measured workloads of the paged 8-bit KV cache: its tables, writes and attention, as a server calls them.

Four kinds of pass:

  tables   a scheduler's step on the GPU: blocks and slots for the new tokens of every request
           (``paged_kv_reserve``), then blocks given back where drafts were rejected or requests ended
           (``paged_kv_trim``)
  write    keys and values of the new tokens quantised into their blocks (``fp8_kv_write``)
  decode   one query token a request over the paged cache (``fp8_paged_decode``)
  attend   several query tokens a request, causal (``fp8_paged_attention``)

The cache holds e4m3 codes [blocks, heads, tokens of a block, D] and one fp32 scale for each block and head, a power of
two where the package wrote it.  Head counts and lengths are those of the repository's benchmark, demo and tests or lie
between them.
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_MOST = 448.0             # the largest e4m3 value
_LOW = -110               # exponent of the scale of a block of zeros


def listed():
    return [
        # A decode step's tables: a request a row, one token each, a few rows idle or of a draft of four.
        dict(name="tables_step", kind="tables", rows=64, least=1, most=4, held=9000, block=64, seed=1),
        # A burst of prompts into small blocks.
        dict(name="tables_prompts", kind="tables", rows=512, least=20, most=2000, held=3000, block=16, seed=2),
        # A decode step's tokens into one layer's cache.
        dict(name="write_step", kind="write", rows=64, least=1, most=1, held=9000, hk=8, d=128, block=64, dtype="bf16", seed=3),
        # Prompts of one prefill batch into one layer's cache.
        dict(name="write_prompts", kind="write", rows=6, least=2000, most=4096, held=1000, hk=8, d=128, block=64, dtype="bf16", seed=4),
        # Chunks at head dim 256, small blocks, fp16.
        dict(name="write_d256_fp16", kind="write", rows=9, least=100, most=700, held=3000, hk=4, d=256, block=32, dtype="fp16", seed=5),
        # One chat request: latency.
        dict(name="decode_one_request", kind="decode", rows=1, low=1021, high=1021, h=32, hk=8, d=128, block=64, dtype="bf16", seed=6),
        # Many requests of all lengths from one token on.
        dict(name="decode_ragged", kind="decode", rows=160, low=1, high=4100, h=8, hk=2, d=128, block=32, dtype="bf16", seed=7),
        # A full serving batch at long context (the benchmark's decode configuration, lengths up to it).
        dict(name="decode_batch_32k", kind="decode", rows=16, low=20000, high=32768, h=32, hk=8, d=128, block=64, dtype="bf16", seed=8),
        # Head dim 256, fp16, smallest blocks.
        dict(name="decode_d256_fp16", kind="decode", rows=24, low=500, high=6007, h=16, hk=4, d=256, block=16, dtype="fp16", seed=9),
        # Verification of short drafts.
        dict(name="attend_drafts", kind="attend", rows=32, most=5, least=5, low=300, high=8190, h=32, hk=8, d=128, block=64, dtype="bf16",
             seed=10),
        # A chunk of a long prompt over what the cache holds of it.
        dict(name="attend_chunk", kind="attend", rows=1, most=2048, least=2048, low=10240, high=10240, h=32, hk=8, d=128, block=64,
             dtype="bf16", seed=11),
        # Chunks and single tokens in one batch at head dim 256, fp16.
        dict(name="attend_mixed_d256", kind="attend", rows=7, most=777, least=0, low=800, high=6007, h=16, hk=4, d=256, block=32,
             dtype="fp16", seed=12),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["tables", "write", "decode", "attend"])
    seed = rng.randrange(1 << 20)
    block = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["bf16", "fp16"])
    d = rng.choice([128, 128, 256])
    hk = rng.choice([1, 2, 4, 8])
    g = rng.choice([1, 2, 3, 4, 7, 8, 16])
    if kind == "tables":
        rows = _log_int(rng, 1, 512)
        return dict(kind=kind, rows=rows, most=_log_int(rng, 1, (1 << 17) // rows * (4 if rows > 16 else 1)), least=1,
                    held=_log_int(rng, 1, 9000), block=block, seed=seed)
    if kind == "write":
        rows = _log_int(rng, 1, 256)
        return dict(kind=kind, rows=rows, most=_log_int(rng, 1, max(1, 12000 // rows)), least=1, held=_log_int(rng, 1, 9000 if rows <= 64 else 2000),
                    hk=hk, d=d, block=block, dtype=rng.choice(["bf16", "fp16", "fp32"]), seed=seed)
    if kind == "decode":
        rows = _log_int(rng, 1, 256)
        high = _log_int(rng, 1, min(131072, (1 << 18) * 12 * 128 // (rows * hk * d)))
        return dict(kind=kind, rows=rows, low=rng.choice([0, 1, high // 2, high]), high=high, h=hk * g, hk=hk, d=d, block=block,
                    dtype=rng.choice(["bf16", "fp16", "bf16", "fp32"]), seed=seed)
    rows = _log_int(rng, 1, 40)
    high = _log_int(rng, 1, 10240 if rows <= 8 else 4000)
    most = _log_int(rng, 1, max(1, min(2048, high, int(7e10 / (rows * hk * g * high * d)))))
    return dict(kind=kind, rows=rows, most=most, least=rng.choice([0, 1, most]), low=max(most, high // 8), high=high, h=hk * g, hk=hk, d=d,
                block=block, dtype=dtype, seed=seed)


# ------------------------------------------------------------------------------------------------ inputs
def _between(gen, n, low, high):
    """n whole numbers of low .. high, spread over their logarithm."""
    lo, hi = math.log(low + 1), math.log(high + 1)
    x = torch.exp(lo + (hi - lo) * torch.rand(n, generator=gen, dtype=torch.float64)).round().long() - 1
    return x.clamp(low, high)


def _lens(case):
    """(tokens held before, new tokens) of every request: sizes belong to the case, not to the seed of its values."""
    gen = torch.Generator().manual_seed(case["seed"])
    rows = case["rows"]
    if case["kind"] in ("tables", "write"):
        held = _between(gen, rows, 0, case["held"])
        new = _between(gen, rows, case["least"], case["most"])
        if case["kind"] == "tables":
            new[torch.rand(rows, generator=gen) < 0.1] = 0
            held[torch.rand(rows, generator=gen) < 0.1] = 0
        return held, new
    total = _between(gen, rows, case["low"], case["high"])
    if case["kind"] == "decode":
        return total, torch.ones_like(total)
    new = torch.minimum(_between(gen, rows, case["least"], case["most"]), total)
    return total - new, new


def _ceil(a, b):
    return (a + b - 1) // b


def _round_codes(x, scale):
    """e4m3 codes of x / scale (a power of two): fp32 in, uint8 out."""
    return (x / scale).clamp(-_MOST, _MOST).to(torch.float8_e4m3fn).view(torch.uint8)


def _scale_of(amax):
    """The smallest power of two that is at least amax / 448, as a float built from its bits."""
    f, x = torch.frexp(amax)
    e = torch.where(f <= 0.875, x - 9, x - 8)
    e = torch.where(amax > 0, e, _LOW).clamp(min=_LOW)
    return ((e.int() + 127) << 23).view(torch.float32)


def _table(gen, held, rows, width, blocks):
    """A block table as a pool leaves it: blocks in no order, -1 where a request holds none; and the blocks left over."""
    order = torch.randperm(blocks, generator=gen).int()
    has = torch.arange(width)[None] < held[:, None]
    table = torch.full((rows, width), -1, dtype=torch.int32)
    table[has] = order[: int(held.sum())]
    return table, order[int(held.sum()):]


def _values(gen, *shape):
    """Activations: normal, eight channels of a larger offset, each token with a size of its own."""
    x = torch.randn(*shape, generator=gen, device="cuda")
    x[..., :8] += 4.0
    return x * torch.exp(0.7 * torch.randn(*shape[:-1], 1, generator=gen, device="cuda"))


def _cache(gen, blocks, hk, block, d):
    x = _values(gen, blocks, hk, block, d)
    scale = _scale_of(x.abs().amax(dim=(2, 3)))
    return _round_codes(x, scale[:, :, None, None]).view(torch.float8_e4m3fn), scale


def prepare(case, seed):
    held, new = _lens(case)
    gen = torch.Generator().manual_seed(seed)
    dev = torch.Generator(device="cuda").manual_seed(seed)
    rows, block = case["rows"], case["block"]
    if case["kind"] in ("decode", "attend"):
        total = held if case["kind"] == "decode" else held + new
    else:
        total = held + new
    width = max(1, int(_ceil(total.max(), block)))
    st = dict(case=case, block=block)
    if case["kind"] == "tables":
        blocks = int(_ceil(total, block).sum()) + 7
        width += 3
        table, free = _table(gen, _ceil(held, block), rows, width, blocks)
        stack = torch.zeros(blocks, dtype=torch.int32)
        stack[: free.numel()] = free
        count = torch.tensor([free.numel()], dtype=torch.int32)
        # the tables of the step before, in one buffer: a pass starts by going back to them
        st["before"] = torch.cat([held.int(), count, stack, table.flatten()]).cuda()
        st["now"] = st["before"].clone()
        parts = st["now"].split([rows, 1, blocks, rows * width])
        st["lengths"], st["count"], st["free"], st["table"] = parts[0], parts[1], parts[2], parts[3].view(rows, width)
        st["new"] = new.int().cuda()
        # what is kept: some drafts are rejected, some requests end
        keep = held + (torch.rand(rows, generator=gen) * (new + 1)).long()
        keep[torch.rand(rows, generator=gen) < 0.15] = 0
        st["keep"] = keep.int().cuda()
        st["slots"] = int(new.sum()) + 5
        return st
    blocks = int(_ceil(total, block).sum()) + 3
    table, _ = _table(gen, _ceil(total, block), rows, width, blocks)
    st["k"], st["ks"] = _cache(dev, blocks, case["hk"], block, case["d"])
    st["v"], st["vs"] = _cache(dev, blocks, case["hk"], block, case["d"])
    dt = _DTYPES[case["dtype"]]
    if case["kind"] == "write":
        tokens = int(new.sum())
        cu = torch.cumsum(new, 0)
        r = torch.repeat_interleave(torch.arange(rows), new)
        p = held[r] + torch.arange(tokens) - (cu - new)[r]
        slots = table[r, p // block].long() * block + p % block
        st["slot_map"] = torch.cat([slots, torch.full((3,), -1)]).cuda()     # a padded batch
        st["key"] = _values(dev, tokens + 3, case["hk"], case["d"]).to(dt)
        st["value"] = _values(dev, tokens + 3, case["hk"], case["d"]).to(dt)
        return st
    st["table"], st["lengths"] = table.cuda(), total.int().cuda()
    st["longest"] = int(total.max())
    st["scaling"] = case["d"] ** -0.5
    if case["kind"] == "decode":
        st["query"] = torch.randn(rows, case["h"], 1, case["d"], generator=dev, device="cuda").to(dt)
    else:
        st["cu"] = torch.cat([torch.zeros(1, dtype=torch.long), torch.cumsum(new, 0)]).int().cuda()
        st["chunk"] = max(1, int(new.max()))
        st["query"] = torch.randn(max(1, int(new.sum())), case["h"], case["d"], generator=dev, device="cuda").to(dt)
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_reserve(st):
    new, lengths, table, free, count, block = st["new"], st["lengths"], st["table"], st["free"], st["count"], st["block"]
    n = new.clamp(min=0)
    had, want = _ceil(lengths, block), _ceil(lengths + n, block)
    need = want - had
    cu = torch.cat([torch.zeros_like(n[:1]), torch.cumsum(n, 0, dtype=torch.int32)])
    off = torch.cumsum(need, 0) - need
    ok = (need.sum() <= count[0]) & (want.max() <= table.shape[1]) & (cu[-1] <= st["slots"])
    j = torch.arange(table.shape[1], device="cuda")[None]
    fresh = (j >= had[:, None]) & (j < want[:, None]) & ok
    at = (count[0] - 1 - (off[:, None] + j - had[:, None])).clamp(0, free.shape[0] - 1)
    table.copy_(torch.where(fresh, free[at], table))
    t = torch.arange(st["slots"], device="cuda")
    r = torch.searchsorted(cu[1:], t.int(), right=True).clamp(max=n.shape[0] - 1)
    p = lengths[r] + t - cu[r]
    valid = (t < cu[-1]) & ok
    b = table[r, (p // block).clamp(0, table.shape[1] - 1)].long()
    slot_map = torch.where(valid, b * block + p % block, -1)
    positions = torch.where(valid, p, 0).int()
    lengths.add_(torch.where(ok, n, 0))
    count.sub_(torch.where(ok, need.sum(), 0).int())
    return slot_map, positions, torch.where(ok, cu, 0), torch.where(ok, 0, 1).int().view(1)


def _plain_trim(st):
    keep, lengths, table, free, count, block = st["keep"], st["lengths"], st["table"], st["free"], st["count"], st["block"]
    to = torch.minimum(keep.clamp(min=0), lengths)
    had, kept = _ceil(lengths, block), _ceil(to, block)
    gone = had - kept
    off = torch.cumsum(gone, 0) - gone
    j = torch.arange(table.shape[1], device="cuda")[None]
    out = (j >= kept[:, None]) & (j < had[:, None])
    at = count[0] + gone.sum() - 1 - (off[:, None] + j - kept[:, None])
    free[at[out]] = table[out]
    table.masked_fill_(out, -1)
    lengths.copy_(to)
    count.add_(gone.sum().int())


def _plain_write(x, slot_map, codes, scale, block):
    keep = slot_map >= 0
    slots, x = slot_map[keep], x[keep].float()
    touched, which = torch.unique(slots // block, return_inverse=True)
    amax = torch.zeros(touched.shape[0], x.shape[1], device="cuda")
    amax.scatter_reduce_(0, which[:, None].expand(-1, x.shape[1]), x.abs().amax(2), "amax")
    first = torch.full_like(touched, block).scatter_reduce_(0, which, slots % block, "amin")
    was = torch.where(first[:, None] > 0, scale[touched], 0.0)
    now = torch.maximum(was, _scale_of(amax))
    old = codes[touched].float() * scale[touched][:, :, None, None]
    old = _round_codes(old, now[:, :, None, None])
    stays = torch.arange(block, device="cuda")[None] < first[:, None]
    raw = codes.view(torch.uint8)
    raw[touched] = torch.where(stays[:, None, :, None], old, raw[touched])
    raw[touched[which], :, slots % block] = _round_codes(x, now[which][:, :, None])
    scale[touched] = now


def _gathered(codes, scale, table, longest, block):
    """[rows, heads, keys, D] values of the blocks that the table names."""
    b = table[:, : _ceil(max(1, longest), block)].clamp(min=0).long()
    x = codes.view(torch.uint8)[b].view(torch.float8_e4m3fn).float() * scale[b][..., None, None]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _plain_rows(q, limit, st):
    """Attention of q [rows, heads, n, D] to the first limit[rows, n] keys of each request."""
    k = _gathered(st["k"], st["ks"], st["table"], st["longest"], st["block"])
    v = _gathered(st["v"], st["vs"], st["table"], st["longest"], st["block"])
    rows, h, n, d = q.shape
    g = h // k.shape[1]
    s = q.float().reshape(rows, k.shape[1], g * n, d) @ k.transpose(2, 3) * st["scaling"]
    seen = torch.arange(k.shape[2], device="cuda")[None, None] < limit.repeat(1, g)[:, :, None]
    s = s.masked_fill_(~seen[:, None], -math.inf)
    m = s.amax(3, keepdim=True).clamp(min=-3e38)
    p = s.sub_(m).exp_()
    total = p.sum(3, keepdim=True)
    v = v.masked_fill_(~seen.any(1)[:, None, :, None], 0.0)
    out = (p @ v) / torch.where(total > 0, total, 1.0)
    lse = m + torch.log(total)
    return out.view(rows, h, n, d), lse.view(rows, h, n)


def _plain_decode(st):
    out, lse = _plain_rows(st["query"], st["lengths"][:, None], st)
    return out.to(st["query"].dtype), lse[:, :, 0]


def _plain_attend(st):
    q, cu, n = st["query"], st["cu"].long(), st["chunk"]
    i = torch.arange(n, device="cuda")[None]
    count = (cu[1:] - cu[:-1])[:, None]
    padded = q[(cu[:-1, None] + i).clamp(max=q.shape[0] - 1)].transpose(1, 2)
    limit = torch.where(i < count, st["lengths"][:, None] - count + 1 + i, 0)
    out, lse = _plain_rows(padded, limit, st)
    t = torch.arange(q.shape[0], device="cuda")
    r = torch.searchsorted(cu[1:], t, right=True).clamp(max=count.shape[0] - 1)
    inside = t < cu[-1]
    out = torch.where(inside[:, None, None], out[r, :, (t - cu[r]).clamp(0, n - 1)], 0.0)
    lse = torch.where(inside[:, None], lse[r, :, (t - cu[r]).clamp(0, n - 1)], -math.inf)
    return out.to(q.dtype), lse


def run(st):
    case = st["case"]
    if case["kind"] == "tables":
        st["now"].copy_(st["before"])
        if own:
            import sageattention_b200.nvfp4 as nv
            step = nv.paged_kv_reserve(st["new"], st["lengths"], st["table"], st["free"], st["count"], st["slots"], st["block"])
            nv.paged_kv_trim(st["keep"], st["lengths"], st["table"], st["free"], st["count"], st["block"])
        else:
            step = _plain_reserve(st)
            _plain_trim(st)
        return [*step, st["lengths"], st["table"], st["free"], st["count"]]
    if case["kind"] == "write":
        if own:
            import sageattention_b200.nvfp4 as nv
            nv.fp8_kv_write(st["key"], st["value"], st["slot_map"], st["k"], st["v"], st["ks"], st["vs"])
        else:
            _plain_write(st["key"], st["slot_map"], st["k"], st["ks"], st["block"])
            _plain_write(st["value"], st["slot_map"], st["v"], st["vs"], st["block"])
        return [st["k"], st["v"], st["ks"], st["vs"]]
    if case["kind"] == "decode":
        if own:
            import sageattention_b200.nvfp4 as nv
            return nv.fp8_paged_decode(st["query"], st["k"], st["v"], st["ks"], st["vs"], st["table"], st["lengths"], st["scaling"],
                                       num_key_value_groups=case["h"] // case["hk"], return_lse=True)
        return _plain_decode(st)
    if own:
        import sageattention_b200.nvfp4 as nv
        return nv.fp8_paged_attention(st["query"], st["cu"], st["k"], st["v"], st["ks"], st["vs"], st["table"], st["lengths"],
                                      st["scaling"], num_key_value_groups=case["h"] // case["hk"], return_lse=True)
    return _plain_attend(st)


def work(case):
    held, new = (x.double() for x in _lens(case))
    block = case["block"]
    if case["kind"] == "tables":
        tokens = float(new.sum())
        fresh = float((_ceil(held + new, block) - _ceil(held, block)).sum())
        # new lengths and lengths in, slots and positions out; fresh blocks out of the stack into the table
        return {"bytes": 12 * tokens + 8 * fresh + 24.0 * case["rows"], "flops": 0}
    if case["kind"] == "write":
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": float(new.sum()) * (2 * case["hk"] * case["d"] * (size + 1) + 8), "flops": 0}
    size = 4 if case["dtype"] == "fp32" else 2
    total = held if case["kind"] == "decode" else held + new
    blocks = float(_ceil(total, block).sum())
    keys = float(total.sum())
    tokens = float(case["rows"]) if case["kind"] == "decode" else float(new.sum())
    seen = keys if case["kind"] == "decode" else float((new * (total - new) + new * (new + 1) / 2).sum())
    moved = keys * 2 * case["hk"] * case["d"] + blocks * (8 * case["hk"] + 4) + tokens * case["h"] * (2 * case["d"] * size + 4)
    return {"bytes": moved, "flops": 4.0 * case["h"] * case["d"] * seen}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _nearest(x):
    """Nearest e4m3 value of x, ties to even, largest 448."""
    size = x.abs().clamp(min=2.0 ** -6)
    step = torch.exp2(torch.floor(torch.log2(size)) - 3)
    step = torch.where(size < step * 8, step / 2, torch.where(size >= step * 16, step * 2, step))
    return (torch.round(x / step) * step).clamp(-_MOST, _MOST)


def _exact_write(x, slots, codes, scale, block):
    """Blocks one after the other, from the definition."""
    codes, scale = codes.double(), scale.double()
    x, slots = x.double()[slots >= 0], slots[slots >= 0]
    cut = [0] + [i for i in range(1, len(slots)) if slots[i] // block != slots[i - 1] // block] + [len(slots)]
    for a, b in zip(cut[:-1], cut[1:]):
        n, at = int(slots[a]) // block, int(slots[a]) % block
        part = x[a:b].transpose(0, 1)                                          # [heads, tokens, D]
        amax = part.abs().amax(dim=(1, 2))
        e = torch.ceil(torch.log2(amax.clamp(min=1e-300) / _MOST))
        e = torch.where(torch.exp2(e - 1) * _MOST >= amax, e - 1, torch.where(torch.exp2(e) * _MOST < amax, e + 1, e)).clamp(min=_LOW)
        now = torch.exp2(e)
        if at > 0:
            now = torch.maximum(now, scale[n])
            codes[n, :, :at] = _nearest(codes[n, :, :at] * (scale[n] / now)[:, None, None])
        codes[n, :, at:at + b - a] = _nearest(part / now[:, None, None])
        scale[n] = now
    return codes, scale


def _exact_rows(q, limit, k, v, scaling):
    """q [heads, n, D], k and v [KV heads, keys, D], token i sees limit[i] keys."""
    hk, g = k.shape[0], q.shape[0] // k.shape[0]
    s = torch.einsum("hgnd,hsd->hgns", q.view(hk, g, *q.shape[1:]), k) * scaling
    s = s.masked_fill(torch.arange(k.shape[1], device="cuda") >= limit[:, None], -math.inf)
    lse = torch.logsumexp(s, 3)
    p = torch.exp(s - torch.where(torch.isfinite(lse), lse, 0.0)[..., None])
    return torch.einsum("hgns,hsd->hgnd", p, v).reshape(q.shape), lse.reshape(q.shape[:2])


def exact(case, seed):
    if case["kind"] == "tables":
        return None                                                            # whole numbers
    held, new = _lens(case)
    if case["kind"] == "write" and int(_ceil(new, case["block"]).sum()) > 4000:
        return None
    if case["kind"] == "attend" and work(case)["flops"] > 6e12:
        return None
    st = prepare(case, seed)
    block = case["block"]
    if case["kind"] == "write":
        slots = st["slot_map"].cpu()
        k, ks = _exact_write(st["key"], slots, st["k"], st["ks"], block)
        v, vs = _exact_write(st["value"], slots, st["v"], st["vs"], block)
        return [k, v, ks, vs]
    decode = case["kind"] == "decode"
    total = held if decode else held + new
    q = st["query"].double()
    out, lse = torch.zeros_like(q), torch.full((q.shape[0], q.shape[1]), -math.inf, dtype=torch.float64, device="cuda")
    at = 0
    for r in range(case["rows"]):
        n, keys = (1 if decode else int(new[r])), int(total[r])
        if n == 0 or keys == 0:
            at += n
            continue
        b = st["table"][r, : _ceil(keys, block)].long()
        k, v = ((c[b].double() * s[b].double()[:, :, None, None]).transpose(0, 1).flatten(1, 2)[:, :keys]
                for c, s in ((st["k"].view(torch.uint8).view(torch.float8_e4m3fn), st["ks"]), (st["v"], st["vs"])))
        limit = keys - n + 1 + torch.arange(n, device="cuda")
        if decode:
            out[r], rows_lse = _exact_rows(q[r], limit, k, v, st["scaling"])
            lse[r] = rows_lse[:, 0]
        else:
            o, rows_lse = _exact_rows(q[at:at + n].transpose(0, 1), limit, k, v, st["scaling"])
            out[at:at + n], lse[at:at + n] = o.transpose(0, 1), rows_lse.T
        at += n
    return out, lse
