"""Paged 8-bit KV cache on the GPU against the 64-bit reference of paged_reference.py: tables and codes exactly, attention
within what its roundings can add up to."""

import math

import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu

_HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _nv():
    import sageattention_b200.nvfp4 as nv
    return nv


def _i32(x):
    return torch.as_tensor(x, dtype=torch.int32).cuda()


# ------------------------------------------------------------------------------------------------ tables
class _Tables:
    """The same state on the GPU and in the reference."""

    def __init__(self, rows, width, blocks, seed=0, wider=0):
        g = torch.Generator().manual_seed(seed)
        free = torch.randperm(blocks, generator=g)
        self.ref = dict(lengths=torch.zeros(rows, dtype=torch.long), table=torch.full((rows, width), -1), free=free.clone(), count=blocks)
        self.lengths, self.free, self.count = _i32([0] * rows), _i32(free), _i32([blocks])
        self.table = torch.full((rows, width + wider), -1, dtype=torch.int32, device="cuda")[:, :width]

    def reserve(self, new, slots, block):
        got = _nv().paged_kv_reserve(_i32(new), self.lengths, self.table, self.free, self.count, slots, block)
        want = R.reserve(new, self.ref, slots, block)
        for a, b in zip(got, want):
            assert a.tolist() == (b if isinstance(b, list) else [b])
        self.same()
        return got

    def trim(self, keep, block):
        _nv().paged_kv_trim(_i32(keep), self.lengths, self.table, self.free, self.count, block)
        R.trim(keep, self.ref, block)
        self.same()

    def same(self):
        assert self.lengths.tolist() == self.ref["lengths"].tolist()
        assert self.table.tolist() == self.ref["table"].tolist()
        n = self.ref["count"]
        assert self.count.tolist() == [n] and self.free[:n].tolist() == self.ref["free"][:n].tolist()


@pytest.mark.parametrize("rows,most,block,seed", [(1, 40, 16, 0), (3, 5, 16, 1), (70, 1, 64, 2), (33, 300, 32, 3), (1030, 9, 16, 4), (2049, 4, 64, 7),
                                                  (4100, 3, 128, 5), (2, 9000, 16, 6)])
def test_steps_of_reservations_and_trims(rows, most, block, seed):
    g = torch.Generator().manual_seed(seed)
    t = _Tables(rows, 3 + 4 * (most // block + 1), rows * (3 + 4 * (most // block + 1)), seed, wider=seed % 2)
    for step in range(5):
        new = torch.randint(-1, most + 1, (rows,), generator=g).tolist()
        t.reserve(new, sum(max(0, n) for n in new) + step, block)
        keep = [int(x) for x in t.ref["lengths"] - torch.randint(-2, most + 1, (rows,), generator=g)]
        t.trim(keep, block)
    t.trim([0] * rows, block)
    assert t.ref["count"] == t.free.numel()


def test_a_step_that_does_not_fit_changes_nothing():
    t = _Tables(4, 3, 7)
    t.reserve([20, 0, 33, 1], 60, 16)
    t.reserve([1, 1, 1, 1], 3, 16)                # too few slots
    t.reserve([0, 49, 0, 0], 60, 16)              # wider than the table
    t.reserve([12, 16, 15, 15], 60, 16)           # one block more than there is
    t.reserve([12, 0, 15, 15], 60, 16)
    t.reserve([0, 0, 0, 0], 0, 16)
    t.trim([-5, 7, 2 ** 31 - 1, 1], 16)


def test_lengths_near_the_largest_do_not_wrap():
    t = _Tables(2, 4, 4)
    t.reserve([2 ** 31 - 1, 2 ** 31 - 1], 10, 16)
    t.reserve([3, 2], 10, 16)


# ------------------------------------------------------------------------------------------------ write
def _rows(shape, seed, dtype):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * torch.exp(2 * torch.randn(*shape[:-1], 1, generator=g))
    return x.to(dtype)


def _empty_cache(blocks, hk, block, d, seed, between=0):
    """Codes and scales with something in them; `between` bytes lie between the blocks."""
    g = torch.Generator().manual_seed(seed)
    flat = torch.randint(0, 256, (blocks, hk * block * d + between), generator=g, dtype=torch.uint8)
    flat[flat == 0x7F] = 0
    flat[flat == 0xFF] = 0
    flat = flat.cuda()
    codes = flat[:, : hk * block * d].unflatten(1, (hk, block, d)).view(torch.float8_e4m3fn)
    scale = torch.exp2(torch.randint(-8, -2, (blocks, hk), generator=g).float()).cuda()
    return codes, scale, flat


def _as_values(codes):
    return codes.contiguous().view(torch.uint8).cpu().view(torch.float8_e4m3fn).double()


def _check_write(key, value, slots, block, d, hk, blocks, between=0):
    k, ks, kflat = _empty_cache(blocks, hk, block, d, 1, between)
    v, vs, vflat = _empty_cache(blocks, hk, block, d, 2, between)
    gaps = kflat[:, hk * block * d:].clone(), vflat[:, hk * block * d:].clone()
    want = []
    for x, c, s in ((key, k, ks), (value, v, vs)):
        cc, ss = _as_values(c), s.cpu().double()
        R.write(x.cpu().double().reshape(-1, hk, d), slots, cc, ss, block)
        want.append((cc, ss))
    _nv().fp8_kv_write(key, value, torch.as_tensor(slots, dtype=torch.int64).cuda(), k, v, ks, vs)
    for (cc, ss), c, s in zip(want, (k, v), (ks, vs)):
        assert torch.equal(s.cpu().double(), ss)
        got = _as_values(c)
        assert torch.equal(torch.isnan(got), torch.isnan(cc))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(cc))
    assert torch.equal(kflat[:, hk * block * d:], gaps[0]) and torch.equal(vflat[:, hk * block * d:], gaps[1])


def _runs(lens, starts, block, seed, blocks):
    """Slots of requests: lens[i] tokens from position starts[i] on, in blocks of no order; -1 in between."""
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).tolist()
    slots = []
    for i, (n, s) in enumerate(zip(lens, starts)):
        mine = [order.pop() for _ in range(-(-(s + n) // block))]
        slots += [mine[p // block] * block + p % block for p in range(s, s + n)]
        if i % 3 == 2:
            slots += [-1, -7]
    return slots


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,block,hk", [(128, 16, 1), (128, 64, 3), (256, 32, 2), (256, 128, 1)])
def test_written_codes_are_the_definitions(dtype, d, block, hk):
    lens = [1, 1, 17, 130, 64, 2, 15, 1, 1, 300]
    starts = [0, 5, 15, 3, 0, 127, 1, 63, 40, 31]
    slots = _runs(lens, starts, block, 3, 100)
    key, value = _rows((len(slots), hk, d), 5, dtype).cuda(), _rows((len(slots), hk, d), 6, dtype).cuda()
    _check_write(key, value, slots, block, d, hk, 100, between=16)


@pytest.mark.parametrize("tokens,hk", [(1, 1), (200, 8), (2500, 4)])
def test_one_token_a_request_and_long_prompts(tokens, hk):
    block = 16
    one = _runs([1] * min(tokens, 200), [i % 40 for i in range(min(tokens, 200))], block, 8, 800)
    long = _runs([tokens], [7], block, 9, 800)
    for slots in (one, long):
        key, value = _rows((len(slots), hk, 128), 15, torch.bfloat16).cuda(), _rows((len(slots), hk, 128), 16, torch.bfloat16).cuda()
        _check_write(key, value, slots, block, 128, hk, 800)


def test_strided_and_unaligned_rows_and_the_decode_shape():
    slots = _runs([3, 20, 1], [14, 0, 9], 16, 2, 30)
    wide = _rows((len(slots), 6, 2, 136), 1, torch.bfloat16).cuda()
    _check_write(wide[:, ::2, 0, :128], wide[:, 1::2, 1, 8:], slots, 16, 128, 3, 30)
    _check_write(wide[:, ::2, 0, 3:131], wide[:, 1::2, 1, 1:129], slots, 16, 128, 3, 30)      # not on 16 bytes
    heads_first = _rows((3, len(slots), 128), 4, torch.float16).cuda().transpose(0, 1)
    _check_write(heads_first, heads_first, slots, 16, 128, 3, 30)
    slots = _runs([1] * 20, [4] * 20, 16, 5, 30)
    one = _rows((len(slots), 3, 1, 128), 7, torch.float16).cuda()
    _check_write(one, one, slots, 16, 128, 3, 30)


def test_skipped_slots_and_values_that_are_not_finite():
    slots = [5 * 16 + 3, -1, 2 * 16, 2 * 16 + 1, 30 * 16, 2 ** 40, 7 * 16 + 15, -2 ** 40]
    key = _rows((8, 2, 128), 1, torch.bfloat16)
    key[[1, 4, 5, 7]] = math.nan                                    # nobody's tokens
    key[3, 0, 5], key[3, 0, 6], key[3, 1, 7] = math.inf, -math.inf, math.nan
    value = torch.zeros(8, 2, 128, dtype=torch.bfloat16)            # blocks of zeros
    value[2, 1, 3] = 3.3e38
    value[6, 0, 0] = 1e-38
    _check_write(key.cuda(), value.cuda(), slots, 16, 128, 2, 30)


def test_no_tokens():
    k, ks, _ = _empty_cache(2, 1, 16, 128, 1)
    before = _as_values(k)
    x = torch.empty(0, 1, 128, dtype=torch.bfloat16, device="cuda")
    _nv().fp8_kv_write(x, x, torch.empty(0, dtype=torch.int64, device="cuda"), k, k.clone(), ks, ks.clone())
    assert torch.equal(_as_values(k), before)


# ------------------------------------------------------------------------------------------------ attention
def _cache(blocks, hk, block, d, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    codes = (torch.randn(blocks, hk, block, d, generator=g) * 60).clamp(-448, 448).to(torch.float8_e4m3fn)
    scale = torch.exp2(torch.randint(-7, -5, (blocks, hk), generator=g).float() + spread * torch.randn(blocks, hk, generator=g).round())
    return codes, scale


def _table(lengths, block, blocks, seed, width=None):
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).tolist()
    width = width or max(1, max(-(-n // block) for n in lengths)) + 1
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    for r, n in enumerate(lengths):
        for j in range(-(-n // block)):
            table[r, j] = order.pop()
    return table


def _spoil(codes, scale, table, lengths, block):
    """NaN codes and scales wherever no request has a key."""
    raw = codes.view(torch.uint8)
    used = torch.zeros(codes.shape[0], block, dtype=torch.bool)
    for r, n in enumerate(lengths):
        for p in range(n):
            if 0 <= table[r, p // block] < codes.shape[0]:
                used[table[r, p // block], p % block] = True
    raw[~used[:, None, :].expand(-1, codes.shape[1], -1)] = 0x7F
    scale[~used.any(1)] = math.nan


def _chunk(dtype, d, tokens, g, requests):
    """Whether a call takes the kernel for many rows."""
    return dtype != torch.float32 and -(-tokens * g // requests) > (32 if d == 128 else 16)


def _key_scales(scale, row, length, block):
    """[Hk, length]: the scale of every key's block."""
    return R.gather(torch.ones(scale.shape[0], scale.shape[1], block, 1), scale, row, length, block)[..., 0]


def _close(got, lse, q, k, v, vscale, limits, scaling, g, hidden=None, chunk=False):
    """Rows of one request.  With A = sum p |v|, S = scaling * sum |q| |k|: scores are off by delta = S (D + 8) 2^-23 (products
    of exact halves summed in fp32; an fp32 q is two halves, 2^-22), a weight by its rounding to halves (2^-11, as two
    2^-22), exp2 and the sums by (keys + 8) 2^-23; the result is rounded once.  Halves end at 2^-24: a weight p vs is held times
    2^5 / W, W = the largest p of 32 keys times their largest vs (at least what a warp's weights are relative to), so its
    rounding is at least 2^-30 W, and with codes of at most 448 a value is off by 2^-30 W 448 keys: all that is left of it
    where the code of the one key that counts is 0.  Calls of many rows (`chunk`) take 128 keys at once and hold weights times 2^3:
    2^-28; and K and V of a block as halves relative to the largest scale of the 128 keys, which below 2^-14 of it are off by
    2^-25 of it: in a score scaling * sum |q| 2^-25 of the largest K scale, in the result 2^-25 sum p of the largest V scale."""
    if hidden is not None:
        k, v = k[:, ~hidden], v[:, ~hidden]
        vscale = torch.where(hidden, 0.0, vscale)
        spread = torch.zeros(vscale.shape[1], dtype=torch.long)
        spread[~hidden] = torch.arange(int((~hidden).sum()))
        limits = [int((~hidden[:max(0, n)]).sum()) for n in limits]
    qd = q.cpu().double()
    want, want_lse = R.attend(qd, k, v, limits, scaling, g)
    size, _ = R.attend(qd, k, v.abs(), limits, scaling, g)
    kk = k.abs().repeat_interleave(g, 0)
    top = torch.einsum("nhd,hsd->nhs", qd.abs(), kk).amax(2) * scaling if k.shape[1] else torch.zeros(want_lse.shape).double()
    two = q.dtype == torch.float32
    delta = top * (q.shape[2] + 8) * 2.0 ** -23 + (k.shape[1] + 8) * 2.0 ** -23 + 2.0 ** -21 * (1 + top)
    tol = size * (2 * delta + (2.0 ** -21 if two else 2.0 ** -11))[..., None] + want.abs() * _HALF_STEP[q.dtype] + 1e-30
    if k.shape[1]:
        kv = k.repeat_interleave(g, 0)
        p = torch.exp(torch.einsum("nhd,hsd->nhs", qd, kv) * scaling - want_lse[..., None])
        p = torch.where(torch.arange(k.shape[1]) < torch.tensor(limits)[:, None, None], p, 0.0)
        if hidden is not None:                                       # keys where they lie, for the groups of 32
            p = torch.where(hidden, 0.0, p[:, :, spread])
        keys = 128 if chunk else 32
        pad = -p.shape[2] % keys
        groups = lambda x: torch.nn.functional.pad(x, (0, pad)).unflatten(-1, (-1, keys)).amax(-1)
        w = (groups(p) * groups(vscale.double()).repeat_interleave(g, 0)).amax(2)
        tol = tol + (2.0 ** (-28 if chunk else -30) * 448 * k.shape[1] * w)[..., None]
        if chunk:
            top_k = qd.abs().sum(2) * scaling * 2.0 ** -25 * float(k.abs().max())     # every block here has codes above 1
            delta = delta + top_k
            tol = tol + (size * 2 * top_k[..., None]) + (2.0 ** -25 * float(vscale.max()))
    if q.dtype == torch.float16:
        tol = tol + 2.0 ** -25                                       # subnormals
    off = (got.cpu().double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())
    if lse is not None:
        none = torch.isinf(want_lse)
        assert torch.equal(torch.isinf(lse.cpu()), none)
        d = (lse.cpu().double() - want_lse)[~none].abs()
        assert bool((d <= (delta + 2.0 ** -22 * want_lse.abs())[~none]).all())


def _decode_case(lengths, h, hk, d, block, dtype, seed=0, spread=2.0, spoil=True, table=None, query=None):
    blocks = sum(-(-n // block) for n in lengths) + 3
    k, ks = _cache(blocks, hk, block, d, seed, spread)
    v, vs = _cache(blocks, hk, block, d, seed + 100, spread)
    table = _table(lengths, block, blocks, seed) if table is None else table
    if spoil:
        _spoil(k, ks, table, lengths, block)
        _spoil(v, vs, table, lengths, block)
    q = torch.randn(len(lengths), h, 1, d, generator=torch.Generator().manual_seed(seed + 7)).to(dtype) if query is None else query
    scaling = d ** -0.5
    out, lse = _nv().fp8_paged_decode(q.cuda(), k.cuda(), v.cuda(), ks.cuda(), vs.cuda(), table.cuda(), _i32(lengths), scaling, h // hk,
                                      return_lse=True)
    assert out.shape == q.shape and out.dtype == dtype and lse.shape == (len(lengths), h)
    for r, n in enumerate(lengths):
        kk, vv = R.gather(k, ks, table[r], n, block), R.gather(v, vs, table[r], n, block)
        _close(out[r].transpose(0, 1), lse[r:r + 1], q[r].transpose(0, 1), kk, vv, _key_scales(vs, table[r], n, block), [n], scaling, h // hk,
               chunk=_chunk(dtype, d, 1, h // hk, 1))
    return out, lse


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("h,hk,d,block", [(4, 1, 128, 16), (8, 2, 128, 64), (16, 1, 256, 32), (3, 3, 256, 128), (7, 1, 128, 32), (40, 2, 128, 16)])
def test_decode_of_ragged_lengths(h, hk, d, block, dtype):
    lengths = [1, 0, 15, 16, 17, 127, 128, 129, 0, 255, 64, 700]
    _decode_case(lengths, h, hk, d, block, dtype, seed=h)


@pytest.mark.parametrize("lengths,hk", [([5000], 1), ([1], 1), ([0], 2), ([3333, 1, 2048], 2), ([40] * 300, 1)])
def test_decode_split_over_the_chip(lengths, hk):
    _decode_case(lengths, 4 * hk, hk, 128, 64, torch.bfloat16, seed=11)


def test_scales_far_apart():
    """V scales from 2^-60 to 2^60 beside each other, and scales that are no powers of two."""
    lengths, block, d = [300, 64, 17], 16, 128
    blocks = sum(-(-n // block) for n in lengths)
    k, ks = _cache(blocks, 2, block, d, 3, 0.0)
    v, vs = _cache(blocks, 2, block, d, 4, 0.0)
    table = _table(lengths, block, blocks, 1)
    g = torch.Generator().manual_seed(9)
    q = torch.randn(3, 8, 1, d, generator=g).to(torch.float16)
    for vscale in (torch.exp2(torch.randint(-60, 60, vs.shape, generator=g).float()), torch.rand(vs.shape, generator=g) * 3e-3 + 1e-5,
                   torch.where(torch.rand(vs.shape, generator=g) < 0.5, 0.0, 2.0 ** -6), torch.full(vs.shape, 2.0 ** -110)):
        kscale = torch.rand(ks.shape, generator=g) * 1e-2
        out, lse = _nv().fp8_paged_decode(q.float().cuda(), k.cuda(), v.cuda(), kscale.cuda(), vscale.cuda(), table.cuda(), _i32(lengths),
                                          d ** -0.5, 4, return_lse=True)
        for r, n in enumerate(lengths):
            kk, vv = R.gather(k, kscale, table[r], n, block), R.gather(v, vscale, table[r], n, block)
            _close(out[r].transpose(0, 1), lse[r:r + 1], q[r].float().transpose(0, 1), kk, vv,
                   _key_scales(vscale, table[r], n, block), [n], d ** -0.5, 4)


def test_table_entries_that_are_no_block_hide_their_keys():
    lengths, block = [100, 33, 40], 16
    blocks = 14
    k, ks = _cache(blocks, 1, block, 128, 3)
    v, vs = _cache(blocks, 1, block, 128, 4)
    table = _table(lengths, block, blocks, 1)
    table[0, 2], table[0, 6], table[1, 0], table[2, :] = -5, 2 ** 31 - 1, 14, -1
    q = torch.randn(3, 4, 1, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    out, lse = _nv().fp8_paged_decode(q.cuda(), k.cuda(), v.cuda(), ks.cuda(), vs.cuda(), table.cuda(), _i32(lengths), 0.1, 4, return_lse=True)
    for r, n in enumerate(lengths):
        bad = torch.tensor([not 0 <= int(table[r, p // block]) < blocks for p in range(n)])
        row = table[r].clamp(0, blocks - 1)
        kk, vv = R.gather(k, ks, row, n, block), R.gather(v, vs, row, n, block)
        _close(out[r].transpose(0, 1), lse[r:r + 1], q[r].transpose(0, 1), kk, vv, _key_scales(vs, row, n, block), [n], 0.1, 4, hidden=bad)
    # lengths that the table cannot hold, or below zero, read nothing outside it
    over = _nv().fp8_paged_decode(q.cuda(), k.cuda(), v.cuda(), ks.cuda(), vs.cuda(), table.cuda(), _i32([2 ** 31 - 1, -3, 40]), 0.1, 4)
    assert torch.equal(over[1], torch.zeros_like(over[1])) and bool(torch.isfinite(over.float()).all())


def test_nan_and_infinite_operands_reach_their_rows_only():
    lengths, block = [50, 50], 16
    k, ks = _cache(8, 1, block, 128, 3)
    v, vs = _cache(8, 1, block, 128, 4)
    table = _table(lengths, block, 8, 1)
    k.view(torch.uint8)[table[0, 1], 0, 3, 5] = 0x7F
    q = torch.randn(2, 4, 1, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    q[1, 2] = math.inf
    out, lse = _nv().fp8_paged_decode(q.cuda(), k.cuda(), v.cuda(), ks.cuda(), vs.cuda(), table.cuda(), _i32(lengths), 0.1, 4, return_lse=True)
    assert bool(torch.isnan(out[0]).all()) and bool(torch.isnan(lse[0]).all())
    assert bool(torch.isnan(out[1, 2]).all())
    assert bool(torch.isfinite(out[1, [0, 1, 3]].float()).all())
    one = _nv().fp8_paged_decode(q[:1].cuda(), k.cuda(), v.cuda(), ks.cuda(), vs.cuda(),
                                 torch.tensor([[int(table[0, 1])]], dtype=torch.int32).cuda(), _i32([4]), 0.1, 4)
    assert bool(torch.isnan(one).all())


def _attend_case(new, held, h, hk, d, block, dtype, seed=0, behind=0, spoil=True, cu=None):
    total = [a + b for a, b in zip(new, held)]
    blocks = sum(-(-n // block) for n in total) + 2
    k, ks = _cache(blocks, hk, block, d, seed)
    v, vs = _cache(blocks, hk, block, d, seed + 50)
    table = _table(total, block, blocks, seed)
    if spoil:
        _spoil(k, ks, table, total, block)
        _spoil(v, vs, table, total, block)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    tokens = starts[-1] + behind
    q = torch.randn(tokens, h, d, generator=torch.Generator().manual_seed(seed + 7)).to(dtype)
    scaling = d ** -0.5
    out, lse = _nv().fp8_paged_attention(q.cuda(), _i32(starts), k.cuda(), v.cuda(), ks.cuda(), vs.cuda(), table.cuda(), _i32(total), scaling,
                                         h // hk, return_lse=True)
    assert out.shape == q.shape and lse.shape == (tokens, h)
    for r, n in enumerate(new):
        if n:
            a, b = starts[r], starts[r + 1]
            kk, vv = R.gather(k, ks, table[r], total[r], block), R.gather(v, vs, table[r], total[r], block)
            _close(out[a:b], lse[a:b], q[a:b], kk, vv, _key_scales(vs, table[r], total[r], block), [held[r] + 1 + i for i in range(n)],
                   scaling, h // hk, chunk=_chunk(dtype, d, tokens, h // hk, len(new)))
    assert bool((out[starts[-1]:] == 0).all()) and bool((lse[starts[-1]:] == -math.inf).all())
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("h,hk,d,block", [(4, 1, 128, 16), (8, 2, 128, 64), (6, 2, 256, 32), (16, 1, 128, 128)])
def test_attention_of_several_tokens_a_request(h, hk, d, block, dtype):
    _attend_case([1, 0, 5, 17, 33, 1, 64], [0, 9, 40, 100, 0, 300, 65], h, hk, d, block, dtype, seed=h, behind=3)


@pytest.mark.parametrize("new,held", [([200], [0]), ([9], [30]), ([17, 9, 20], [200, 5, 0]), ([130], [700]), ([257, 1, 1, 300], [5, 900, 0, 129])])
@pytest.mark.parametrize("d", [128, 256])
def test_chunks_of_prompts(new, held, d):
    _attend_case(new, held, 8, 2, d, 32, torch.bfloat16, seed=3)


@pytest.mark.parametrize("h,hk,d,most,dtype", [(32, 8, 128, 8, torch.bfloat16), (32, 8, 128, 30, torch.float16), (16, 2, 128, 20, torch.bfloat16),
                                               (16, 4, 256, 8, torch.float16), (32, 8, 128, 5, torch.bfloat16), (32, 8, 128, 4, torch.float32)])
def test_long_shares_of_every_kernel(h, hk, d, most, dtype):
    """So much work that a CTA goes through many key tiles of a unit and through several units; a few requests are compared."""
    g = torch.Generator().manual_seed(h + most)
    block, requests = 64, 50
    new = torch.randint(1, most + 1, (requests,), generator=g).tolist()
    new[3], new[7] = most, 1                                           # on average above most / 2
    held = torch.randint(1500, 4000, (requests,), generator=g).tolist()
    total = [a + b for a, b in zip(new, held)]
    blocks = sum(-(-n // block) for n in total) + 1
    k, ks = _cache(blocks, hk, block, d, 1)
    v, vs = _cache(blocks, hk, block, d, 2)
    table = _table(total, block, blocks, 3)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = torch.randn(starts[-1], h, d, generator=g).to(dtype)
    scaling = d ** -0.5
    out, lse = _nv().fp8_paged_attention(q.cuda(), _i32(starts), k.cuda(), v.cuda(), ks.cuda(), vs.cuda(), table.cuda(), _i32(total), scaling,
                                         h // hk, return_lse=True)
    for r in (0, 3, 7, 20, 33, 49):
        a, b = starts[r], starts[r + 1]
        kk, vv = R.gather(k, ks, table[r], total[r], block), R.gather(v, vs, table[r], total[r], block)
        _close(out[a:b], lse[a:b], q[a:b], kk, vv, _key_scales(vs, table[r], total[r], block), [held[r] + 1 + i for i in range(new[r])],
               scaling, h // hk, chunk=_chunk(dtype, d, starts[-1], h // hk, requests))


def test_single_tokens_are_decode():
    """The same rows through both entries, to the bit: one schedule."""
    lengths, block = [33, 500, 1, 0, 90], 16
    blocks = 50
    k, ks = _cache(blocks, 2, block, 128, 3)
    v, vs = _cache(blocks, 2, block, 128, 4)
    table = _table(lengths, block, blocks, 1)
    q = torch.randn(5, 8, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    args = (k.cuda(), v.cuda(), ks.cuda(), vs.cuda(), table.cuda(), _i32(lengths), 0.1, 4)
    a = _nv().fp8_paged_attention(q, _i32(range(6)), *args)
    b = _nv().fp8_paged_decode(q[:, :, None], *args)
    assert torch.equal(a, b[:, :, 0])


def test_more_tokens_than_keys_and_bad_offsets_stay_inside():
    block = 16
    k, ks = _cache(4, 1, block, 128, 3)
    v, vs = _cache(4, 1, block, 128, 4)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32)
    q = torch.randn(12, 4, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    args = (k.cuda(), v.cuda(), ks.cuda(), vs.cuda(), table.cuda())
    out, lse = _nv().fp8_paged_attention(q.cuda(), _i32([0, 6, 12]), *args, _i32([4, 20]), 0.1, 4, return_lse=True)
    assert bool((out[:2] == 0).all()) and bool((lse[:2] == -math.inf).all())
    kk, vv = R.gather(k, ks, table[0], 4, block), R.gather(v, vs, table[0], 4, block)
    _close(out[:6], lse[:6], q[:6], kk, vv, _key_scales(vs, table[0], 4, block), [-1, 0, 1, 2, 3, 4], 0.1, 4)
    for cu in ([0, 100, 200], [-5, 6, 12], [8, 3, 12], [12, 12, 12], [3, 6, 9], [2 ** 31 - 1, -2 ** 31, 0]):
        out = _nv().fp8_paged_attention(q.cuda(), _i32(cu), *args, _i32([4, 20]), 0.1, 4)
    torch.cuda.synchronize()


def test_same_bits_every_time_and_strided_operands():
    lengths, block = [33, 500, 1, 0, 90], 16
    k, ks = _cache(100, 2, block, 128, 3)
    v, vs = _cache(100, 2, block, 128, 4)
    table = _table(lengths, block, 100, 1, width=64).cuda()
    q = torch.randn(5, 8, 1, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    both = torch.stack([k.cuda(), v.cuda()], 1)                       # K and V of a block beside each other
    scales = torch.stack([ks.cuda(), vs.cuda()], 1)
    plain = [_nv().fp8_paged_decode(q, k.cuda(), v.cuda(), ks.cuda(), vs.cuda(), table, _i32(lengths), 0.1, 4) for _ in range(3)]
    other = _nv().fp8_paged_decode(torch.stack([q, q], 4)[..., 0], both[:, 0], both[:, 1], scales[:, 0], scales[:, 1], table[:, :40],
                                   _i32(lengths), 0.1, 4)
    heads = _nv().fp8_paged_decode(q.transpose(0, 1).contiguous().transpose(0, 1), both[:, 0], both[:, 1], scales[:, 0], scales[:, 1],
                                   table[:, :40], _i32(lengths), 0.1, 4)
    for x in (*plain[1:], other, heads):
        assert torch.equal(x, plain[0])


# ------------------------------------------------------------------------------------------------ together
def _server(dtype, capture):
    """Prompts, then steps of one token each with a request that ends and one that comes, two layers; every attention is
    compared with the reference on the cache's own contents, and the contents with the reference's writes."""
    nv = _nv()
    h, hk, d, block, rows = 8, 2, 128, 16, 4
    cache = nv.FP8PagedKVCache(2, 40, hk, d, rows, 160, "cuda", block_size=block)
    g = torch.Generator().manual_seed(5)
    ref = [[torch.zeros(40, hk, block, d).double(), torch.zeros(40, hk).double()] for _ in range(4)]
    lengths = [0] * rows

    def step(new, inputs):
        out = []
        s = cache.reserve(new, inputs[0][0].shape[0])
        for layer, (key, value, query) in enumerate(inputs):
            cache.write(layer, key, value, s.slot_map)
            out.append(cache.attend(layer, query, s.cu_seqlens, d ** -0.5, h // hk, return_lse=True))
        return s, out

    def check(new, inputs, s, out):
        assert s.shortage.tolist() == [0]
        for r in range(rows):
            lengths[r] += new[r]
        assert cache.lengths.tolist() == lengths
        table, slots = cache.block_table.cpu(), s.slot_map.tolist()
        for layer, (key, value, query) in enumerate(inputs):
            for x, c, sc, (rc, rs) in ((key, cache.k, cache.k_scale, ref[2 * layer]), (value, cache.v, cache.v_scale, ref[2 * layer + 1])):
                R.write(x.cpu().double(), slots, rc, rs, block)
                for r in range(rows):
                    assert torch.equal(R.gather(c[layer].cpu(), sc[layer].cpu(), table[r], lengths[r], block),
                                       R.gather(rc, rs, table[r], lengths[r], block))
            at = 0
            for r, n in enumerate(new):
                if n:
                    kk, vv = (R.gather(*ref[2 * layer + i], table[r], lengths[r], block) for i in (0, 1))
                    _close(out[layer][0][at:at + n], out[layer][1][at:at + n], query[at:at + n], kk, vv,
                           _key_scales(ref[2 * layer + 1][1], table[r], lengths[r], block), [lengths[r] - n + 1 + i for i in range(n)],
                           d ** -0.5, h // hk, chunk=_chunk(dtype, d, query.shape[0], h // hk, rows))
                    at += n

    def inputs_of(n):
        mk = lambda heads: (torch.randn(n, heads, d, generator=g) * 2).to(dtype).cuda()
        return [(mk(hk), mk(hk), mk(h)) for _ in range(2)]

    def end(keep):
        for r, n in enumerate(keep):
            lengths[r] = min(lengths[r], n)
        cache.trim(_i32(keep))

    new = [37, 0, 100, 5]
    inputs = inputs_of(sum(new) + 2)
    check(new, inputs, *step(_i32(new), inputs))
    graph, static = None, None
    for i in range(24):
        new = [1, 0 if i < 3 else 1, 1, 0 if i in (4, 5) else 1]
        inputs = inputs_of(rows)
        if not capture:
            result = step(_i32(new), inputs)
        else:
            if graph is None:
                static = (_i32([0] * rows), inputs_of(rows))
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    step(*static)                                     # no new token: the state stays
                torch.cuda.current_stream().wait_stream(side)
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    result_static = step(*static)
            static[0].copy_(_i32(new))
            for a, b in zip(static[1], inputs):
                for x, y in zip(a, b):
                    x.copy_(y)
            graph.replay()
            result = result_static
        check(new, inputs, *result)
        if i == 8:
            end([10 ** 6, 2, 0, lengths[3] - 3])
    end([0] * rows)
    assert cache.free_count.tolist() == [40] and sorted(cache.free_blocks.tolist()) == list(range(40))
    assert bool((cache.block_table == -1).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_server_of_several_requests(dtype):
    _server(dtype, capture=False)


def test_the_same_steps_replayed_from_a_graph():
    _server(torch.bfloat16, capture=True)


def test_two_captured_decodes_replayed_in_turn_and_on_other_streams():
    lengths, block = [333, 50], 16
    graphs, outs, want = [], [], []
    for seed in (1, 2):
        k, ks = (x.cuda() for x in _cache(40, 1, block, 128, seed))
        v, vs = (x.cuda() for x in _cache(40, 1, block, 128, seed + 10))
        table = _table(lengths, block, 40, seed).cuda()
        q = torch.randn(2, 4, 1, 128, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()
        n = _i32(lengths)
        call = lambda q=q, k=k, v=v, ks=ks, vs=vs, table=table, n=n: _nv().fp8_paged_decode(q, k, v, ks, vs, table, n, 0.1, 4)
        want.append(call().clone())
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            assert torch.equal(call(), want[-1])
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call())
        graphs.append((graph, call))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for (graph, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


# several tokens a request, one set for each kernel: 8, 16, 24 and more query rows
_KERNELS = [([1, 1, 1], torch.bfloat16, 128), ([2, 3, 2], torch.float16, 128), ([5, 6, 5], torch.bfloat16, 128),
            ([7, 40, 150], torch.bfloat16, 128), ([7, 40, 150], torch.float16, 256), ([5, 6, 5], torch.float32, 256)]


def _set(new, dtype, d, seed, h=8, hk=2, block=16, held=(90, 0, 21)):
    """Operands on the GPU of a batch whose requests have `new` tokens behind `held` others."""
    total = [a + b for a, b in zip(new, held)]
    blocks = sum(-(-n // block) for n in total) + 2
    k, ks = _cache(blocks, hk, block, d, seed)
    v, vs = _cache(blocks, hk, block, d, seed + 50)
    table = _table(total, block, blocks, seed)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = torch.randn(starts[-1], h, d, generator=torch.Generator().manual_seed(seed + 7)).to(dtype)
    cache = [x.cuda() for x in (k, v, ks, vs, table)]
    return q.cuda(), _i32(starts), cache, _i32(total), (k, v, ks, vs, table, total, block)


@pytest.mark.parametrize("new,dtype,d", _KERNELS)
def test_scaling_of_zero_and_below(new, dtype, d):
    q, cu, cache, lengths, (k, v, ks, vs, table, total, block) = _set(new, dtype, d, 1)
    call = lambda q, s: _nv().fp8_paged_attention(q, cu, *cache, lengths, s, 4, return_lse=True)
    for a, b in zip(call(q, -0.1), call(-q, 0.1)):
        assert torch.equal(a, b)
    out, lse = call(q, 0.0)                                            # the mean of what a row sees
    for r, n in enumerate(new):
        a = int(cu[r])
        kk, vv = R.gather(k, ks, table[r], total[r], block), R.gather(v, vs, table[r], total[r], block)
        _close(out[a:a + n], lse[a:a + n], q[a:a + n].cpu(), kk, vv, _key_scales(vs, table[r], total[r], block),
               [total[r] - n + 1 + i for i in range(n)], 0.0, 4, chunk=_chunk(dtype, d, q.shape[0], 4, 3))


@pytest.mark.parametrize("new,dtype,d", _KERNELS)
def test_attention_of_rows_that_are_not_aligned(new, dtype, d):
    q, cu, cache, lengths, _ = _set(new, dtype, d, 2)
    want = _nv().fp8_paged_attention(q, cu, *cache, lengths, 0.1, 4)
    flat = torch.empty(q.numel() + 1, dtype=dtype, device="cuda")[1:].view(q.shape)
    flat.copy_(q)
    wide = torch.empty(q.shape[0], 8, d + 3, dtype=dtype, device="cuda")[..., :d]
    wide.copy_(q)
    last = torch.empty(d, 8, q.shape[0], dtype=dtype, device="cuda").permute(2, 1, 0)
    last.copy_(q)
    for x in (flat, wide, last):
        assert torch.equal(_nv().fp8_paged_attention(x, cu, *cache, lengths, 0.1, 4), want)


@pytest.mark.parametrize("new,dtype,d", _KERNELS)
def test_two_captured_batches_replayed_at_once(new, dtype, d):
    graphs, outs, want = [], [], []
    for seed in (1, 2):
        q, cu, cache, lengths, _ = _set(new, dtype, d, seed)
        call = lambda q=q, cu=cu, cache=cache, lengths=lengths: _nv().fp8_paged_attention(q, cu, *cache, lengths, 0.1, 4)
        want.append(call().clone())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call())
        graphs.append((graph, call))                                   # the operands live as long as the graph
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for (graph, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


@pytest.mark.parametrize("tokens", [20, 3000])
def test_a_block_named_twice_spoils_no_other(tokens):
    """Its codes are anybody's; those of the call's other blocks, and of blocks that it does not name, are as ever."""
    block, blocks = 16, 400
    slots = torch.arange(tokens) + 3 * block
    twice = slots.clone()
    twice[tokens // 2 // block * block] = 5                            # inside block 0, as the last token is
    twice[-1] = 5
    key, value = _rows((tokens, 2, 128), 1, torch.bfloat16).cuda(), _rows((tokens, 2, 128), 2, torch.bfloat16).cuda()
    got = []
    for s in (slots, twice):
        codes = [torch.zeros(blocks, 2, block, 128, dtype=torch.uint8, device="cuda") for _ in range(2)]
        scales = [torch.zeros(blocks, 2, device="cuda") for _ in range(2)]
        _nv().fp8_kv_write(key, value, s.cuda(), *codes, *scales)
        got.append((codes, scales))
    touched = {0} | {int(s) // block for s, t in zip(slots, twice) if s != t}
    others = torch.tensor([b for b in range(blocks) if b not in touched]).cuda()
    for a, b in zip(sum(map(list, got[0]), []), sum(map(list, got[1]), [])):
        assert torch.equal(a[others], b[others])


def test_registered_operators_are_the_same_calls():
    import sageattention_b200.nvfp4.custom_ops  # noqa: F401
    ns, nv = torch.ops.sageattention_b200, _nv()
    a, b = (nv.FP8PagedKVCache(1, 12, 2, 128, 3, 64, "cuda", block_size=16) for _ in range(2))
    new = _i32([5, 0, 20])
    step = a.reserve(new, 27)
    got = ns.paged_kv_reserve(new, b.lengths, b.block_table, b.free_blocks, b.free_count, 27, 16)
    for x, y in zip(step, got):
        assert torch.equal(x, y)
    key, value = _rows((27, 2, 128), 1, torch.bfloat16).cuda(), _rows((27, 2, 128), 2, torch.bfloat16).cuda()
    a.write(0, key, value, step.slot_map)
    ns.fp8_kv_write(key, value, got[0], b.k[0], b.v[0], b.k_scale[0], b.v_scale[0])
    q = _rows((27, 8, 128), 3, torch.bfloat16).cuda()
    for x, y in zip(a.attend(0, q, step.cu_seqlens, 0.1, 4, True),
                    ns.fp8_paged_attention(q, got[2], b.k[0], b.v[0], b.k_scale[0], b.v_scale[0], b.block_table, b.lengths, 0.1, 4)):
        assert torch.equal(x, y)
    for x, y in zip(a.decode(0, q[:3, :, None], 0.1, 4, True),
                    ns.fp8_paged_decode(q[:3, :, None], b.k[0], b.v[0], b.k_scale[0], b.v_scale[0], b.block_table, b.lengths, 0.1, 4)):
        assert torch.equal(x, y)
    a.trim(_i32([1, 0, 17]))
    ns.paged_kv_trim(_i32([1, 0, 17]), b.lengths, b.block_table, b.free_blocks, b.free_count, 16)
    assert torch.equal(a.block_table, b.block_table) and torch.equal(a.free_blocks, b.free_blocks) and torch.equal(a.lengths, b.lengths)


def test_positions_feed_the_rotary_pack():
    """A step's positions are what ``rope_quant_nvfp4`` takes."""
    nv = _nv()
    cache = nv.FP8PagedKVCache(1, 12, 1, 128, 2, 64, "cuda", block_size=16)
    cache.reserve(_i32([7, 30]), 37)
    step = cache.reserve(_i32([2, 1]), 5)
    assert step.positions.tolist() == [7, 8, 30, 0, 0]
    ang = torch.arange(64, device="cuda")[:, None] * 0.01 * torch.arange(64, device="cuda")[None]
    x = _rows((1, 5, 128), 3, torch.bfloat16).cuda()
    packed = nv.rope_quant_nvfp4(x, ang.cos(), ang.sin(), positions=step.positions)
    one = nv.rope_quant_nvfp4(x[:, 2:3], ang.cos(), ang.sin(), pos0=30)
    assert torch.equal(packed[0][:, 2], one[0][:, 0])


def test_the_demo_runs_with_the_paged_cache():
    from sageattention_b200 import _lib
    from sageattention_b200.nvfp4 import demo_decode
    rep = demo_decode.main(["--layers", "2", "--hidden", "512", "--heads", "4", "--kv-heads", "2", "--vocab", "512", "--batch", "2",
                            "--prompt", "150", "--new", "4", "--window", "64"])
    assert math.isfinite(rep["fp8"]["logit_cos"])
    assert rep["fp8"]["bytes"] == 2 * 2 * 2 * 3 * 2 * (64 * 128 + 4)      # layers, K and V, requests, blocks, heads
    assert _lib.read_status("cuda:0") == 0


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    nv = _nv()
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    k = torch.zeros(4, 2, 16, 128, device="cuda").to(torch.float8_e4m3fn)
    s = torch.ones(4, 2, device="cuda")
    x = torch.zeros(3, 2, 128, dtype=torch.bfloat16, device="cuda")
    slots = torch.zeros(3, dtype=torch.int64, device="cuda")
    bad_write = [
        (TypeError, (x, x.half(), slots, k, k, s, s)), (TypeError, (x.int(), x.int(), slots, k, k, s, s)),
        (AssertionError, (x, x[:2], slots, k, k, s, s)), (AssertionError, (x[:, :1], x[:, :1], slots, k, k, s, s)),
        (TypeError, (x, x, slots.int(), k, k, s, s)), (AssertionError, (x, x, slots[:2], k, k, s, s)),
        (AssertionError, (x, x, slots, k, k[:2], s, s)), (AssertionError, (x, x, slots, k, k, s[:2], s)),
        (TypeError, (x, x, slots, k.float(), k, s, s)), (TypeError, (x, x, slots, k, k, s.half(), s)),
        (AssertionError, (x, x, slots, k[:, :, :8], k[:, :, :8], s, s)), (AssertionError, (x, x, slots, k[..., :64], k[..., :64], s, s)),
        (ValueError, (x, x, slots, k[0], k[0], s, s)), (ValueError, (x[0], x[0], slots, k, k, s, s)),
        (AssertionError, (x, x, slots, k[:1].expand(4, -1, -1, -1), k, s, s)), (RuntimeError, (x, x.cpu(), slots, k, k, s, s)),
        (RuntimeError, (x, x, slots.cpu(), k, k, s, s)),
    ]
    for err, args in bad_write:
        with pytest.raises(err):
            nv.fp8_kv_write(*args)
    q, table, n = torch.zeros(3, 4, 1, 128, dtype=torch.bfloat16, device="cuda"), i(3, 2), i(3)
    ok = (q, k, k, s, s, table, n, 0.1, 2)
    nv.fp8_paged_decode(*ok)
    for err, at, what in [(AssertionError, 0, q[:2]), (AssertionError, 0, q.expand(-1, -1, 2, -1)), (ValueError, 0, q[0]),
                          (TypeError, 0, q.double()), (AssertionError, 0, q[..., :64]), (AssertionError, 8, 4), (AssertionError, 8, 0),
                          (TypeError, 5, table.long()), (ValueError, 5, table[0]), (AssertionError, 5, table[:1].expand(3, -1)),
                          (AssertionError, 6, n[:2]), (TypeError, 6, n.long()), (RuntimeError, 6, n.cpu()), (AssertionError, 6, i(6)[::2])]:
        args = list(ok)
        args[at] = what
        with pytest.raises(err):
            nv.fp8_paged_decode(*args)
    qt = torch.zeros(5, 4, 128, dtype=torch.bfloat16, device="cuda")
    for err, cu, query in [(AssertionError, i(3), qt), (TypeError, i(4).long(), qt), (ValueError, i(4), q), (ValueError, None, qt)]:
        with pytest.raises(err):
            nv.fp8_paged_attention(query, cu, k, k, s, s, table, n, 0.1, 2)
    good = [i(3), i(3), i(3, 2), i(8), i(1)]
    for at, what, err in [(0, i(2), AssertionError), (1, i(3).long(), TypeError), (2, i(3, 0), AssertionError), (3, i(8).float(), TypeError),
                          (4, i(2), AssertionError), (2, i(2, 3).t(), AssertionError)]:
        args = list(good)
        args[at] = what
        with pytest.raises(err):
            nv.paged_kv_reserve(*args, 4, 16)
        with pytest.raises(err):
            nv.paged_kv_trim(*args, 16)
    with pytest.raises(RuntimeError, match="block_size"):
        nv.paged_kv_reserve(*good, 4, 24)
    with pytest.raises(AssertionError):
        nv.paged_kv_reserve(*good, -1, 16)


# ------------------------------------------------------------------------------------------------ padding
def _padded(front, behind, dtype, d, h=32, hk=8, requests=32, held=200):
    """A captured step's batch: one token for each request, and thousands of rows that are nobody's around them."""
    q, _, cache, lengths, _ = _set([1] * requests, dtype, d, 3, h=h, hk=hk, held=[held] * requests)
    cu = _i32([front + i for i in range(requests + 1)])
    rows = torch.randn(front + requests + behind, h, d, device="cuda").to(dtype)
    rows[front:front + requests] = q
    return rows, cu, cache, lengths


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 256), (torch.float32, 128)])
@pytest.mark.parametrize("front,behind", [(0, 3000), (3000, 0), (1501, 777)])
def test_thousands_of_padded_rows_are_zeros(front, behind, dtype, d):
    rows, cu, cache, lengths = _padded(front, behind, dtype, d)
    out, lse = _nv().fp8_paged_attention(rows, cu, *cache, lengths, 0.1, 4, return_lse=True)
    want, want_lse = _nv().fp8_paged_decode(rows[front:front + 32, :, None], *cache, lengths, 0.1, 4, return_lse=True)
    for x, y in ((slice(0, front), 0), (slice(front + 32, None), 0)):
        assert bool((out[x] == y).all()) and bool((lse[x] == -math.inf).all())
    # the other kernel, maybe: weights and the result rounded apart
    size = float(want.float().abs().max())
    assert float((out[front:front + 32].float() - want[:, :, 0].float()).abs().max()) <= size * 4 * _HALF_STEP[torch.bfloat16]
    assert float((lse[front:front + 32] - want_lse).abs().max()) <= 1e-3


def test_padded_rows_are_cleared_by_the_whole_chip():
    """8160 padded rows, 67 MB: at most what the call takes without them, the few rows through the kernel for many, and ten plain fills of as
    many bytes.  (By one block of threads it was a hundred.)"""
    def time_of(f):
        f()
        times = []
        for _ in range(7):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            torch.cuda.synchronize()
            a.record()
            f()
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return sorted(times)[3]

    rows, cu, cache, lengths = _padded(0, 8160, torch.bfloat16, 128)
    call = lambda rows: time_of(lambda: _nv().fp8_paged_attention(rows, cu, *cache, lengths, 0.1, 4))
    fill = time_of(lambda: torch.zeros_like(rows))
    few, padded = call(rows[:32]), call(rows)
    assert padded <= 4 * few + 10 * fill
