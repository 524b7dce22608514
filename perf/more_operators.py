"""Measured workloads of decoding with drafted trees over the paged 8-bit KV cache, and of what prepares its queries and keys.

Five kinds of pass:

  tree     what the nodes of every request's tree see, and where they stand (``draft_tree``), then their attention over the
           paged cache (``fp8_paged_tree_attention``)
  verify   which drafted tokens the target's probabilities keep, from given random numbers, and the token that comes next
           (``verify_drafts``)
  keep     keys and values of the accepted path moved together in all layers of the cache (``paged_kv_keep_path``)
  norm     RMS norm of every head's queries and keys, then their rotation by position (``qk_norm_rope``)
  train    the same with the gradients of both operands and both weights

A request's tokens are its tree: the first one is the token that the step before ended with, every other one names its
parent among those in front of it.  The cache holds e4m3 codes [blocks, heads, tokens of a block, D] and one fp32 scale for
each block and head.  Head counts and lengths are those of the repository's benchmark, demo and tests or lie between them.
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_MOST = 448.0             # the largest e4m3 value
_LOW = -110               # exponent of the scale of a block of zeros


def listed():
    return [
        # One chat request with a tree of eight: latency.
        dict(name="tree_one_request", kind="tree", rows=1, least=8, most=8, low=1021, high=1021, h=32, hk=8, d=128, block=64, dtype="bf16", seed=1),
        # A serving batch: trees of 16 to 64 nodes over contexts of all lengths.
        dict(name="tree_batch", kind="tree", rows=32, least=16, most=64, low=300, high=8190, h=32, hk=8, d=128, block=64, dtype="bf16", seed=2),
        # Small trees at head dim 256, smallest blocks, fp16.
        dict(name="tree_d256_fp16", kind="tree", rows=12, least=3, most=26, low=500, high=6007, h=16, hk=4, d=256, block=16, dtype="fp16", seed=3),
        # Chains of five drawn from a draft model's probabilities.
        dict(name="verify_chains", kind="verify", rows=32, least=6, most=6, vocab=32000, drawn=True, branch=1, dtype="fp32", seed=4),
        # Trees of the likeliest tokens, which no draft probabilities belong to, over a large vocabulary.
        dict(name="verify_likeliest", kind="verify", rows=64, least=26, most=26, vocab=131072, drawn=False, branch=4, dtype="fp32", seed=5),
        # Trees with several draws a node, a vocabulary whose rows begin anywhere.
        dict(name="verify_drawn_trees", kind="verify", rows=7, least=2, most=21, vocab=50001, drawn=True, branch=3, dtype="bf16", seed=6),
        # The demo's small model: latency.
        dict(name="keep_step", kind="keep", rows=2, least=8, most=8, held=2048, layers=4, hk=2, d=128, block=64, seed=7),
        # A serving batch, paths that end in other blocks than they lie in.
        dict(name="keep_batch", kind="keep", rows=64, least=16, most=64, held=400, layers=16, hk=8, d=128, block=16, seed=8),
        # A decode step of a batch, operands as the fused projection leaves them: latency.
        dict(name="norm_step", kind="norm", z=1, s=32, h=32, hk=8, d=128, layout="thd", dtype="bf16", weights="bf16", seed=9),
        # Prompts of one prefill batch.
        dict(name="norm_prompts", kind="norm", z=1, s=16001, h=32, hk=8, d=128, layout="thd", dtype="bf16", weights="bf16", seed=10),
        # Training at head dim 256, an odd length, fp16 with weights in fp32.
        dict(name="train_d256_fp16", kind="train", z=3, s=1237, h=16, hk=4, d=256, layout="zhsd", dtype="fp16", weights="fp32", seed=11),
        # A training step of the benchmark's heads.
        dict(name="train_step", kind="train", z=4, s=4096, h=32, hk=8, d=128, layout="zhsd", dtype="bf16", weights="bf16", seed=12),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["tree", "verify", "keep", "norm", "train"])
    seed = rng.randrange(1 << 20)
    block = rng.choice([16, 32, 64, 128])
    d = rng.choice([128, 128, 256])
    hk = rng.choice([1, 2, 4, 8])
    g = rng.choice([1, 2, 3, 4, 7, 8])
    if kind == "tree":
        rows = _log_int(rng, 1, 64)
        most = _log_int(rng, 1, min(64, 2048 // rows))
        high = _log_int(rng, max(2, most), min(16384, max(256, min(int(4e10 / (rows * most * hk * g * d * 4)), int(8e7 / (rows * hk * d))))))
        return dict(kind=kind, rows=rows, least=rng.choice([0, 1, most]), most=most, low=min(high, max(most, high // 8)), high=high, h=hk * g, hk=hk, d=d,
                    block=block, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), seed=seed)
    if kind == "verify":
        rows = _log_int(rng, 1, 128)
        most = _log_int(rng, 1, 64)
        drawn = rng.random() < 0.5
        vocab = _log_int(rng, 100, min(150000, 8000000 // rows, int(2e8 / (rows * most * (2 if drawn else 1)))))
        return dict(kind=kind, rows=rows, least=rng.choice([0, 1, most]), most=most, vocab=vocab, drawn=drawn, branch=rng.choice([1, 2, 4]),
                    dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]), seed=seed)
    if kind == "keep":
        rows = _log_int(rng, 1, 128)
        most = _log_int(rng, 1, 64)
        held = _log_int(rng, 1, 600)
        layers = _log_int(rng, 1, max(1, min(32, int(2.5e8 / (rows * (held + most + block) * hk * d)))))
        return dict(kind=kind, rows=rows, least=rng.choice([0, 1, most]), most=most, held=held, layers=layers, hk=hk, d=d, block=block, seed=seed)
    z = rng.choice([1, 1, 2, 3])
    s = _log_int(rng, 1, int(8e7 / (z * hk * (g + 1) * d)))
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    return dict(kind=kind, z=z, s=s, h=hk * g, hk=hk, d=d, layout=rng.choice(["thd", "zhsd"]) if z == 1 else "zhsd", dtype=dtype,
                weights=rng.choice([dtype, "fp32"]), seed=seed)


# ------------------------------------------------------------------------------------------------ inputs
def _between(gen, n, low, high):
    """n whole numbers of low .. high, spread over their logarithm."""
    lo, hi = math.log(low + 1), math.log(high + 1)
    x = torch.exp(lo + (hi - lo) * torch.rand(n, generator=gen, dtype=torch.float64)).round().long() - 1
    return x.clamp(low, high)


def _ceil(a, b):
    return (a + b - 1) // b


def _sizes(case):
    """(tokens held before, nodes) of every request: sizes belong to the case, not to the seed of its values."""
    gen = torch.Generator().manual_seed(case["seed"])
    rows = case["rows"]
    nodes = _between(gen, rows, case["least"], case["most"])
    nodes[-1] += nodes.sum() == 0                                              # a call has a token at least
    if case["kind"] == "tree":
        total = torch.maximum(_between(gen, rows, case["low"], case["high"]), nodes)
        return total - nodes, nodes
    if case["kind"] == "keep":
        return _between(gen, rows, 0, case["held"]), nodes
    return torch.zeros_like(nodes), nodes


def _parents(gen, nodes, branch):
    """Trees: node i hangs on one of the nodes in front of it, mostly a near one; [sum of nodes] int32, -1 for the first."""
    n = int(nodes.sum())
    i = torch.arange(n) - torch.repeat_interleave(torch.cumsum(nodes, 0) - nodes, nodes)
    if branch == 1:
        return (i - 1).int()
    back = 1 + (torch.rand(n, generator=gen) ** 2 * (2 * branch)).long()
    return torch.where(i == 0, -1, (i - back).clamp(min=0)).int()


def _cu(nodes):
    return torch.cat([torch.zeros(1, dtype=torch.long), torch.cumsum(nodes, 0)]).int()


def _round_codes(x, scale):
    """e4m3 codes of x / scale (a power of two): fp32 in."""
    return (x / scale).clamp(-_MOST, _MOST).to(torch.float8_e4m3fn)


def _scale_of(amax):
    """The smallest power of two that is at least amax / 448, as a float built from its bits."""
    f, x = torch.frexp(amax)
    e = torch.where(f <= 0.875, x - 9, x - 8)
    e = torch.where(amax > 0, e, _LOW).clamp(min=_LOW)
    return ((e.int() + 127) << 23).view(torch.float32)


def _table(gen, held, rows, width, blocks):
    """A block table as a pool leaves it: blocks in no order, -1 where a request holds none."""
    order = torch.randperm(blocks, generator=gen).int()
    has = torch.arange(width)[None] < held[:, None]
    table = torch.full((rows, width), -1, dtype=torch.int32)
    table[has] = order[: int(held.sum())]
    return table


def _values(gen, *shape):
    """Activations: normal, eight channels of a larger offset, each token with a size of its own."""
    x = torch.randn(*shape, generator=gen, device="cuda")
    x[..., :8] += 4.0
    return x * torch.exp(0.7 * torch.randn(*shape[:-1], 1, generator=gen, device="cuda"))


def _cache(gen, *shape):
    """Codes [..., heads, tokens of a block, D] and their scales [..., heads]."""
    x = _values(gen, *shape)
    scale = _scale_of(x.abs().amax(dim=(-2, -1)))
    return _round_codes(x, scale[..., None, None]), scale


def _path_of(gen, parents, nodes):
    """A path down every tree, as a verification leaves it: node numbers request by request, -1 behind; and their count."""
    accepted, count = [], []
    for par in parents.split(nodes.tolist()):
        path = [0] if len(par) else []
        while path and torch.rand(1, generator=gen).item() < 0.8:
            below = (par == path[-1]).nonzero().flatten().tolist()
            if not below:
                break
            path.append(below[int(torch.randint(len(below), (1,), generator=gen))])
        accepted += path + [-1] * (len(par) - len(path))
        count.append(len(path))
    return torch.tensor(accepted, dtype=torch.int32), torch.tensor(count, dtype=torch.int32)


def _prepare_verify(case, st, nodes, gen, dev):
    """Target rows as a softmax gives them, peaked and with a long tail; drafts that mostly agree."""
    t, vocab, dt = int(nodes.sum()), case["vocab"], _DTYPES[case["dtype"]]
    start = torch.repeat_interleave(torch.cumsum(nodes, 0) - nodes, nodes)
    above = (start + st["parents_host"].clamp(min=0)).cuda()
    hang = (start + st["parents_host"])[st["parents_host"] >= 0]
    st["kids"] = int(hang.bincount().max()) if len(hang) else 0                # most children of a node
    logits = torch.randn(t, vocab, generator=dev, device="cuda").mul_(2.0)
    logits.scatter_add_(1, torch.randint(vocab, (t, 6), generator=dev, device="cuda"), 6.0 + 4.0 * torch.rand(t, 6, generator=dev, device="cuda"))
    noise = torch.randn(t, vocab, generator=dev, device="cuda").mul_(0.4).add_(logits)
    st["target"] = torch.softmax(logits, 1).to(dt)
    if case["drawn"]:
        st["draft"] = torch.softmax(noise, 1).to(dt)
        # one draw of its parent's row for every node: the token whose exponential clock is first
        clock = torch.empty(t, vocab, device="cuda").exponential_(generator=dev)
        st["tokens"] = torch.argmax(st["draft"][above].float() / clock, 1)
    else:
        st["draft"] = None
        i = torch.arange(t) - start
        rank = ((st["parents_host"][None] == st["parents_host"][:, None]) & (start[None] == start[:, None]) & (i[None] < i[:, None])).sum(1)
        top = torch.topk(noise, min(vocab, int(rank.max()) + 1), 1).indices
        st["tokens"] = top[above, rank.clamp(max=top.shape[1] - 1).cuda()]
    st["uniforms"] = torch.rand(t, generator=dev, device="cuda")


def _prepare_norm(case, gen, dev):
    z, s, h, hk, d, dt = case["z"], case["s"], case["h"], case["hk"], case["d"], _DTYPES[case["dtype"]]
    st = dict(eps=1e-6)
    heads = h + hk + (hk if case["layout"] == "thd" else 0)                    # the fused projection's values lie behind
    x = _values(dev, z * s, heads, d).to(dt)
    if case["layout"] == "thd":
        st["q"], st["k"] = x[:, :h], x[:, h:h + hk]
        longest = max(40000, s)
        st["positions"] = torch.randint(longest, (s,), generator=gen).int().cuda() if s < 64 else (torch.arange(s) + longest - s).int().cuda()
    else:
        st["q"], st["k"] = (x[:, a:b].contiguous().view(z, s, b - a, d).transpose(1, 2) for a, b in ((0, h), (h, h + hk)))
        longest = s
        st["positions"] = torch.arange(s, dtype=torch.int32, device="cuda")
    angle = torch.arange(longest, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
    st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
    st["wq"], st["wk"] = (1.0 + 0.3 * torch.randn(2, d, generator=dev, device="cuda")).to(_DTYPES[case["weights"]])
    if case["kind"] == "train":
        st["dq"] = torch.randn(z * s, h, d, generator=dev, device="cuda").to(dt)
        st["dk"] = torch.randn(z * s, hk, d, generator=dev, device="cuda").to(dt)
        if case["layout"] == "zhsd":
            st["dq"], st["dk"] = (g.view(z, s, -1, d).transpose(1, 2) for g in (st["dq"], st["dk"]))
        st["leaves"] = [st[n].detach().requires_grad_(True) for n in ("q", "k", "wq", "wk")]
    return st


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    dev = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] in ("norm", "train"):
        return dict(_prepare_norm(case, gen, dev), case=case)
    held, nodes = _sizes(case)
    st = dict(case=case, rows=case["rows"])
    st["parents_host"] = _parents(gen, nodes, case.get("branch", 3))
    st["parents"], st["cu"] = st["parents_host"].cuda(), _cu(nodes).cuda()
    st["most"] = max(1, case["most"])
    if case["kind"] == "verify":
        _prepare_verify(case, st, nodes, gen, dev)
        return st
    total, block, rows = held + nodes, case["block"], case["rows"]
    st["block"] = block
    blocks = int(_ceil(total, block).sum()) + 3
    width = max(1, int(_ceil(total.max(), block)))
    st["table"] = _table(gen, _ceil(total, block), rows, width, blocks).cuda()
    st["lengths"] = total.int().cuda()
    if case["kind"] == "keep":
        st["k"], st["ks"] = _cache(dev, case["layers"], blocks, case["hk"], block, case["d"])
        st["v"], st["vs"] = _cache(dev, case["layers"], blocks, case["hk"], block, case["d"])
        accepted, count = _path_of(gen, st["parents_host"], nodes)
        st["accepted"], st["count"] = accepted.cuda(), count.cuda()
        return st
    st["k"], st["ks"] = _cache(dev, blocks, case["hk"], block, case["d"])
    st["v"], st["vs"] = _cache(dev, blocks, case["hk"], block, case["d"])
    st["longest"], st["scaling"] = int(total.max()), case["d"] ** -0.5
    st["query"] = torch.randn(int(nodes.sum()), case["h"], case["d"], generator=dev, device="cuda").to(_DTYPES[case["dtype"]])
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _padded(st):
    """(token of request r's node i, there is one, parent of it or -1), each [rows, most]."""
    cu, n = st["cu"].long(), st["most"]
    i = torch.arange(n, device="cuda")[None]
    there = i < (cu[1:] - cu[:-1])[:, None]
    at = (cu[:-1, None] + i).clamp(max=st["parents"].shape[0] - 1)
    par = st["parents"][at].long()
    return at, there, torch.where(there & (par >= 0) & (par < i), par, -1)


def _ancestors(par):
    """[rows, n, n]: node j is i or above it."""
    n = par.shape[1]
    up = torch.eye(n, dtype=torch.float64, device="cuda") + (par[:, :, None] == torch.arange(n, device="cuda")).double()
    return torch.linalg.matrix_power(up, n) > 0.5


def _of_tokens(cu, n, values, fill):
    """[T] of [rows, most]: row by row, `fill` where no request is."""
    t = torch.arange(n, device="cuda")
    r = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=cu.shape[0] - 2)
    x = values[r, (t - cu[r]).clamp(0, values.shape[1] - 1)]
    return torch.where((t < cu[-1]).view(-1, *[1] * (x.dim() - 1)), x, fill)


def _plain_tables(st):
    at, there, par = _padded(st)
    seen = _ancestors(par) & there[:, :, None]
    cu = st["cu"].long()
    depth = seen.sum(2) - 1
    pos = (st["lengths"] - (cu[1:] - cu[:-1]))[:, None] + depth
    n, words = seen.shape[1], _ceil(seen.shape[1], 64)
    bits = torch.nn.functional.pad(seen, (0, words * 64 - n)).view(*seen.shape[:2], words, 64).long()
    mask = (bits << torch.arange(64, device="cuda")).sum(3)
    tokens = st["parents"].shape[0]
    return _of_tokens(cu, tokens, mask, 0), _of_tokens(cu, tokens, pos, 0).int()


def _gathered(codes, scale, table, longest, block):
    """[rows, heads, keys, D] values of the blocks that the table names."""
    b = table[:, : _ceil(max(1, longest), block)].clamp(min=0).long()
    x = codes.view(torch.uint8)[b].view(torch.float8_e4m3fn).float() * scale[b][..., None, None]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _plain_attend(st, mask):
    at, there, _ = _padded(st)
    cu, d = st["cu"].long(), st["query"].shape[2]
    q = st["query"][at].float().transpose(1, 2)                                # [rows, heads, n, D]
    k = _gathered(st["k"], st["ks"], st["table"], st["longest"], st["block"])
    v = _gathered(st["v"], st["vs"], st["table"], st["longest"], st["block"])
    rows, h, n, _ = q.shape
    hk, g = k.shape[1], h // k.shape[1]
    context = st["lengths"].long() - (cu[1:] - cu[:-1])
    j = torch.arange(k.shape[2], device="cuda")[None] - context[:, None]       # number of the node that a key is of
    inside = (j < st["lengths"][:, None] - context[:, None]) & there.any(1)[:, None]
    node = j.clamp(min=0)
    word = torch.gather(mask[at], 2, (node // 64).clamp(max=mask.shape[1] - 1)[:, None].expand(-1, n, -1))
    seen = ((word >> (node % 64)[:, None]) & 1).bool() & (node < 64 * mask.shape[1])[:, None]
    seen = (seen | (j < 0)[:, None]) & inside[:, None] & there[:, :, None]
    s = q.reshape(rows, hk, g * n, d) @ k.transpose(2, 3) * st["scaling"]
    s = s.view(rows, hk, g, n, -1).masked_fill_(~seen[:, None, None], -math.inf)
    m = s.amax(4, keepdim=True).clamp(min=-3e38)
    p = s.sub_(m).exp_()
    total = p.sum(4, keepdim=True)
    v = v.masked_fill_(~seen.any(1)[:, None, :, None], 0.0)
    out = (p.view(rows, hk, g * n, -1) @ v).view(rows, hk, g, n, d) / torch.where(total > 0, total, 1.0)
    lse = (m + torch.log(total)).view(rows, h, n)
    t = st["query"].shape[0]
    out = _of_tokens(cu, t, out.reshape(rows, h, n, d).transpose(1, 2), 0.0)
    return out.to(st["query"].dtype), _of_tokens(cu, t, lse.transpose(1, 2), -math.inf)


def _plain_verify(st):
    """Every node's test is of its parent's row and of the siblings in front of it, whatever the path: all at once."""
    at, there, par = _padded(st)
    rows, n = par.shape
    cu, vocab = st["cu"].long(), st["target"].shape[1]
    tok, u = st["tokens"][at], st["uniforms"][at].double()
    i = torch.arange(n, device="cuda")
    before = (par[:, :, None] == par[:, None, :]) & (par >= 0)[:, :, None] & (i[None, :] < i[:, None])     # sibling j in front of i
    above = torch.gather(at, 1, par.clamp(min=0))                              # token of the parent
    p = st["target"].double()
    known = (tok >= 0) & (tok < vocab)
    if st["draft"] is None:
        again = (before & (tok[:, :, None] == tok[:, None, :])).any(2)
        px = torch.where(known & ~again, p[above, tok.clamp(0, vocab - 1)], 0.0)
        mass = (1.0 - (before.double() @ px[:, :, None])[:, :, 0]).clamp(min=0.0)
        passes = u * mass < px
        left = None
    else:
        q = st["draft"].double()
        rank, kids = before.sum(2), (par[:, None, :] == i[:, None]).sum(2)     # number among the siblings; children of a node
        per_row = torch.zeros(p.shape[0], dtype=torch.long, device="cuda").index_put_((at[there],), kids[there])
        now, left, mass = p, p, torch.ones(p.shape[0], dtype=torch.float64, device="cuda")
        passes = torch.zeros_like(known)
        x = tok.clamp(0, vocab - 1)
        for k in range(st["kids"]):
            ok = known & (u * q[above, x] * mass[above] < now[above, x])
            passes = torch.where((rank == k) & (par >= 0), ok, passes)
            now = (now / torch.where(mass > 0, mass, 1.0)[:, None] - q).clamp(min=0.0) * (mass > 0)[:, None]
            mass = now.sum(1)
            left = torch.where((k < per_row)[:, None], now, left)
    chosen = passes & (par >= 0) & ~(before & passes[:, None, :]).any(2)
    up = _ancestors(par)
    path = there & up[:, :, 0] & (~up | (chosen | (i == 0))[:, None, :]).all(2)
    count = path.sum(1)
    order = torch.sort(torch.where(path, i, n), 1).values
    last = (count - 1).clamp(min=0)
    last = torch.gather(order, 1, last[:, None]).clamp(max=n - 1)
    row = torch.gather(at, 1, last)[:, 0]
    if left is None:
        below = torch.where((par == last) & known, tok, vocab)
        rest = torch.nn.functional.pad(p[row], (0, 1)).scatter(1, below, 0.0)[:, :vocab]
    else:
        rest = left[row]
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, p[row])
    upto = torch.cumsum(rest, 1)
    w = st["uniforms"][cu[:-1].clamp(max=st["uniforms"].shape[0] - 1)].double()
    following = (upto <= w[:, None] * upto[:, -1:]).sum(1)
    most = torch.where(rest > 0, torch.arange(vocab, device="cuda"), 0).amax(1)
    following = torch.where(there[:, 0], torch.minimum(following, most), -1)
    t = st["parents"].shape[0]
    return _of_tokens(cu, t, torch.where(order < n, order, -1), -1).int(), torch.where(there[:, 0], count, 0).int(), following


def _plain_keep(st):
    """Every source is read before anything is written."""
    cu, block, lengths = st["cu"].long(), st["block"], st["lengths"].long()
    nodes, count = cu[1:] - cu[:-1], st["count"].long()
    at, there, _ = _padded(dict(st, parents=st["accepted"]))
    j = torch.arange(at.shape[1], device="cuda")[None]
    a = st["accepted"][at].long()
    r, to = ((j < count[:, None]) & (a > j) & there).nonzero(as_tuple=True)    # the tokens that move
    a = a[r, to]
    context = lengths - nodes
    src, dst = context[r] + a, context[r] + to
    from_b, to_b = (st["table"][r, x // block].long() for x in (src, dst))
    touched, which = torch.unique(to_b, return_inverse=True)
    first = torch.full_like(touched, block).scatter_reduce_(0, which, dst % block, "amin")
    return [_plain_move(st[c], st[s], from_b, src % block, touched, which, dst % block, first) for c, s in (("k", "ks"), ("v", "vs"))], \
        (lengths - nodes + count).int()


def _plain_move(codes, scale, from_b, from_o, touched, which, to_o, first):
    """Tokens of all layers and heads from their blocks into others, whose scales grow where they have to."""
    raw = codes.view(torch.uint8)
    x = raw[:, from_b, :, from_o].view(torch.float8_e4m3fn).float()            # [moved, layers, heads, D]
    xs, was = scale[:, from_b].transpose(0, 1), scale[:, touched].transpose(0, 1)
    larger = xs > was[which]
    amax = torch.zeros_like(was).scatter_reduce_(0, which[:, None, None].expand_as(larger),
                                                 torch.where(larger, x.abs().amax(3) * xs, 0.0), "amax")
    now = torch.where(amax > 0, torch.maximum(was, _scale_of(amax)), was)
    old = raw[:, touched].view(torch.float8_e4m3fn).float().transpose(0, 1)    # [touched, layers, heads, tokens, D]
    stays = torch.arange(codes.shape[3], device="cuda")[None] < first[:, None]
    again = _round_codes(old * was[..., None, None], now[..., None, None]).view(torch.uint8)
    again = torch.where(stays[:, None, None, :, None], again, old.to(torch.float8_e4m3fn).view(torch.uint8))
    moved = _round_codes(x * xs[..., None], now[which][..., None]).view(torch.uint8)
    raw[:, touched] = again.transpose(0, 1)
    raw[:, touched[which], :, to_o] = moved
    scale[:, touched] = now.transpose(0, 1)


def _turned(x, c, s):
    """Half-split rotation: element i with element i + D / 2."""
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _by_position(st):
    c, s = st["cos"][st["positions"].long()], st["sin"][st["positions"].long()]
    return (c[:, None], s[:, None]) if st["q"].dim() == 3 else (c, s)


def _plain_norm(x, w, c, s, eps):
    x = x.detach().float()
    return _turned(x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.detach().float(), c, s)


def _plain_norm_grads(x, w, g, c, s, eps):
    x, w = x.detach().float(), w.detach().float()
    inv = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    n, g = x * inv, _turned(g.float(), c, -s)
    gw = g * w
    return inv * (gw - n * (gw * n).mean(-1, keepdim=True)), (g * n).flatten(0, -2).sum(0)


def run(st):
    case = st["case"]
    if case["kind"] == "tree":
        if own:
            import sageattention_b200.nvfp4 as nv
            mask, positions = nv.draft_tree(st["parents"], st["cu"], st["lengths"], st["most"])
            out, lse = nv.fp8_paged_tree_attention(st["query"], st["cu"], mask, st["k"], st["v"], st["ks"], st["vs"], st["table"], st["lengths"],
                                                   st["scaling"], num_key_value_groups=case["h"] // case["hk"], return_lse=True)
        else:
            mask, positions = _plain_tables(st)
            out, lse = _plain_attend(st, mask)
        return [mask, positions, out, lse]
    if case["kind"] == "verify":
        if own:
            import sageattention_b200.nvfp4 as nv
            return [*nv.verify_drafts(st["target"], st["tokens"], st["parents"], st["cu"], st["uniforms"], draft_probs=st["draft"])]
        return [*_plain_verify(st)]
    if case["kind"] == "keep":
        if own:
            import sageattention_b200.nvfp4 as nv
            kept = nv.paged_kv_keep_path(st["accepted"], st["count"], st["cu"], st["lengths"], st["table"], st["k"], st["v"], st["ks"], st["vs"])
        else:
            _, kept = _plain_keep(st)
        return [kept, st["k"], st["v"], st["ks"], st["vs"]]
    if case["kind"] == "norm":
        if own:
            import sageattention_b200.nvfp4 as nv
            return [*nv.qk_norm_rope(st["q"], st["k"], st["wq"], st["wk"], st["cos"], st["sin"], st["positions"], eps=st["eps"])]
        c, s = _by_position(st)
        return [_plain_norm(st[x], st[w], c, s, st["eps"]).to(st[x].dtype) for x, w in (("q", "wq"), ("k", "wk"))]
    if own:
        import sageattention_b200.nvfp4 as nv
        outs = nv.qk_norm_rope(*st["leaves"], st["cos"], st["sin"], st["positions"], eps=st["eps"])
        return [*(x.detach() for x in outs), *torch.autograd.grad(outs, st["leaves"], (st["dq"], st["dk"]))]
    c, s = _by_position(st)
    q, k, wq, wk = st["leaves"]
    outs = [_plain_norm(x, w, c, s, st["eps"]).to(x.dtype) for x, w in ((q, wq), (k, wk))]
    (gq, gwq), (gk, gwk) = (_plain_norm_grads(x, w, g, c, s, st["eps"]) for x, w, g in ((q, wq, st["dq"]), (k, wk, st["dk"])))
    return [*outs, gq.to(q.dtype), gk.to(k.dtype), gwq.to(wq.dtype), gwk.to(wk.dtype)]


def work(case):
    if case["kind"] in ("norm", "train"):
        size, wsize = 4 if case["dtype"] == "fp32" else 2, 4 if case["weights"] == "fp32" else 2
        tokens, heads, d = case["z"] * case["s"], case["h"] + case["hk"], case["d"]
        values, table = float(tokens * heads * d), float((tokens if case["layout"] == "thd" else case["s"]) * (4 * d + 4))
        # operands read, results written; for gradients operands and incoming gradients read, gradients written
        passes = 2 if case["kind"] == "norm" else 5
        return {"bytes": passes * values * size + table + 2.0 * d * wsize * (1 if case["kind"] == "norm" else 2),
                "flops": values * (8 if case["kind"] == "norm" else 28)}
    held, nodes = (x.double() for x in _sizes(case))
    total, tokens, rows = held + nodes, float(nodes.sum()), case["rows"]
    if case["kind"] == "verify":
        size = 4 if case["dtype"] == "fp32" else 2
        both = 2 if case["drawn"] else 1
        # a row of the target's for every request (and of the draft's), of other rows a value each; tokens, parents, numbers in, results out
        asked = float((nodes > 0).sum())
        return {"bytes": asked * case["vocab"] * size * both + tokens * (both * size + 20) + 16.0 * rows, "flops": asked * case["vocab"] * (2 * both)}
    if case["kind"] == "keep":
        # half of a path's tokens move, about: a few of every tree, whose depth is at most its nodes
        moved = float(torch.clamp(nodes - 1, min=0).clamp(max=4).sum()) / 2
        return {"bytes": moved * 4 * case["layers"] * case["hk"] * case["d"] + tokens * 4 + 16.0 * rows + moved * 8 * case["layers"] * case["hk"], "flops": 0}
    size, block = 4 if case["dtype"] == "fp32" else 2, case["block"]
    live = (nodes > 0).double()
    keys, blocks = float((total * live).sum()), float((_ceil(total, block) * live).sum())
    words = _ceil(max(1, case["most"]), 64)
    moved = keys * 2 * case["hk"] * case["d"] + blocks * (8 * case["hk"] + 4) + tokens * (case["h"] * (2 * case["d"] * size + 4) + 8 + 8 * words)
    seen = float((nodes * (held + torch.log2(nodes + 1))).sum())               # a node sees the context and its own path
    return {"bytes": moved, "flops": 4.0 * case["h"] * case["d"] * seen}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _nearest(x):
    """Nearest e4m3 value of x, ties to even, largest 448."""
    size = x.abs().clamp(min=2.0 ** -6)
    step = torch.exp2(torch.floor(torch.log2(size)) - 3)
    step = torch.where(size < step * 8, step / 2, torch.where(size >= step * 16, step * 2, step))
    return (torch.round(x / step) * step).clamp(-_MOST, _MOST)


def _walk_up(parents):
    """[n, n] of one tree, node by node."""
    seen = torch.zeros(len(parents), len(parents), dtype=torch.bool)
    for i, p in enumerate(parents.tolist()):
        if 0 <= p < i:
            seen[i] = seen[p]
        seen[i, i] = True
    return seen


def _exact_tree(case, st, held, nodes):
    q = st["query"].double()
    hk, block = case["hk"], case["block"]
    out, lse = torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    at = 0
    for r, par in enumerate(st["parents_host"].split(nodes.tolist())):
        n, before = len(par), int(held[r])
        if n == 0:
            continue
        b = st["table"][r, : _ceil(before + n, block)].long()
        k, v = ((c.view(torch.uint8)[b].view(torch.float8_e4m3fn).double() * s[b].double()[:, :, None, None]).transpose(0, 1).flatten(1, 2)[:, :before + n]
                for c, s in ((st["k"], st["ks"]), (st["v"], st["vs"])))
        seen = torch.cat([torch.ones(n, before, dtype=torch.bool), _walk_up(par)], 1).cuda()
        x = q[at:at + n].transpose(0, 1).reshape(hk, -1, n, q.shape[2])
        s = (torch.einsum("hgnd,hsd->hgns", x, k) * st["scaling"]).masked_fill(~seen, -math.inf)
        lse[at:at + n] = torch.logsumexp(s, 3).flatten(0, 1).T
        out[at:at + n] = torch.einsum("hgns,hsd->hgnd", torch.softmax(s, 3), v).flatten(0, 1).transpose(0, 1)
        at += n
    return [None, None, out, lse]


def _exact_keep(case, st, held, nodes):
    """Token by token, from the definition."""
    block, table = case["block"], st["table"].cpu()
    values = []
    for codes, scale in ((st["k"], st["ks"]), (st["v"], st["vs"])):
        x, s = codes.view(torch.uint8).view(torch.float8_e4m3fn).double(), scale.double()
        new_x, new_s = x.clone(), s.clone()
        for r, path in enumerate(st["accepted"].cpu().split(nodes.tolist())):
            path = path[: int(st["count"][r])].tolist()
            base = int(held[r])
            into = {}                                                          # block of the table -> [(its offset, source)]
            for j, a in enumerate(path):
                if a != j:
                    into.setdefault((base + j) // block, []).append(((base + j) % block, base + a))
            for t, moves in into.items():
                b = int(table[r, t])
                now, first = s[:, b], moves[0][0]
                for _, src in moves:
                    sb = int(table[r, src // block])
                    amax = x[:, sb, :, src % block].abs().amax(2) * s[:, sb]
                    e = torch.ceil(torch.log2(amax.clamp(min=1e-300) / _MOST))
                    e = torch.where(torch.exp2(e - 1) * _MOST >= amax, e - 1, torch.where(torch.exp2(e) * _MOST < amax, e + 1, e)).clamp(min=_LOW)
                    now = torch.where((s[:, sb] > s[:, b]) & (amax > 0), torch.maximum(now, torch.exp2(e)), now)
                new_x[:, b, :, :first] = _nearest(x[:, b, :, :first] * (s[:, b] / now)[:, :, None, None])
                for o, src in moves:
                    sb = int(table[r, src // block])
                    new_x[:, b, :, o] = _nearest(x[:, sb, :, src % block] * (s[:, sb] / now)[:, :, None])
                new_s[:, b] = now
        values.append((new_x, new_s))
    (k, ks), (v, vs) = values
    return [None, k, v, ks, vs]


def _exact_norm(case, st):
    def turn(x, sign):
        c, s = (t.double()[st["positions"].long()] for t in (st["cos"], st["sin"]))
        if x.dim() == 3:
            c, s = c[:, None], s[:, None]
        h = x.shape[-1] // 2
        y = torch.empty_like(x)
        y[..., :h] = x[..., :h] * c - sign * x[..., h:] * s
        y[..., h:] = x[..., h:] * c + sign * x[..., :h] * s
        return y

    outs, grads, weights = [], [], []
    for x, w, g in (("q", "wq", "dq"), ("k", "wk", "dk")):
        x, w = st[x].detach().double(), st[w].detach().double()
        root = torch.sqrt((x * x).mean(-1, keepdim=True) + st["eps"])
        outs.append(turn(x / root * w, 1.0))
        if case["kind"] == "train":
            g = turn(st[g].double(), -1.0)
            weights.append((g * x / root).reshape(-1, x.shape[-1]).sum(0))
            g = g * w / root
            grads.append(g - x * (g * x).sum(-1, keepdim=True) / (x.shape[-1] * root * root))
    return [*outs, *grads, *weights]


def exact(case, seed):
    if case["kind"] == "verify":
        return None                                                            # whole numbers
    st = prepare(case, seed)
    if case["kind"] in ("norm", "train"):
        return _exact_norm(case, st)
    held, nodes = _sizes(case)
    if case["kind"] == "keep":
        return _exact_keep(case, st, held, nodes)
    return _exact_tree(case, st, held, nodes)
