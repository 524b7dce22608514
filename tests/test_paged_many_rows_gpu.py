"""The kernel for many query rows over the paged 8-bit KV cache where other tests use the one for few: hidden table entries, more
tokens than keys, wide groups, operands that are not finite."""

import math

import pytest
import torch

import paged_reference as R
from test_paged_cache_gpu import _cache, _chunk, _close, _decode_case, _i32, _key_scales, _nv, _spoil, _table

pytestmark = pytest.mark.gpu

# new tokens of three requests (4 query rows each), D, type: one group of 128 rows, two, and at D 256
_MANY = [([20, 9, 12], 128, torch.bfloat16), ([60, 0, 40], 128, torch.float16), ([11, 40, 7], 256, torch.bfloat16), ([50, 1, 33], 256, torch.float16)]


def _batch(new, total, d, dtype, block, seed, hk=2):
    blocks = sum(-(-n // block) for n in total) + 2
    k, ks = _cache(blocks, hk, block, d, seed)
    v, vs = _cache(blocks, hk, block, d, seed + 50)
    table = _table(total, block, blocks, seed)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = torch.randn(starts[-1], 4 * hk, d, generator=torch.Generator().manual_seed(seed + 7)).to(dtype)
    assert _chunk(dtype, d, starts[-1], 4, len(new))
    return k, ks, v, vs, table, starts, q


def _call(q, starts, k, ks, v, vs, table, total, scaling):
    return _nv().fp8_paged_attention(q.cuda(), _i32(starts), k.cuda(), v.cuda(), ks.cuda(), vs.cuda(), table.cuda(), _i32(total), scaling, 4,
                                     return_lse=True)


@pytest.mark.parametrize("block", [16, 64])
@pytest.mark.parametrize("new,d,dtype", _MANY)
def test_table_entries_that_are_no_block_hide_their_keys(new, d, dtype, block):
    total = [300, 130, 70]
    k, ks, v, vs, table, starts, q = _batch(new, total, d, dtype, block, 3)
    blocks = k.shape[0]
    table[0, 1], table[0, 3], table[1, 0], table[2, :] = -5, 2 ** 31 - 1, blocks, -1
    _spoil(k, ks, table, total, block)
    _spoil(v, vs, table, total, block)
    out, lse = _call(q, starts, k, ks, v, vs, table, total, 0.1)
    for r, n in enumerate(new):
        if n == 0:
            continue
        a, b = starts[r], starts[r + 1]
        bad = torch.tensor([not 0 <= int(table[r, p // block]) < blocks for p in range(total[r])])
        row = table[r].clamp(0, blocks - 1)
        kk, vv = (torch.nan_to_num(R.gather(c, s, row, total[r], block)) for c, s in ((k, ks), (v, vs)))
        scales = torch.nan_to_num(_key_scales(vs, row, total[r], block))
        limits = [total[r] - n + 1 + i for i in range(n)]
        _close(out[a:b], lse[a:b], q[a:b], kk, vv, scales, limits, 0.1, 4, hidden=bad, chunk=True)


@pytest.mark.parametrize("new,d,dtype", _MANY)
def test_more_tokens_than_keys(new, d, dtype):
    """A request's first tokens see nothing: zeros and -inf."""
    total, block = [3, 1, 33], 16
    k, ks, v, vs, table, starts, q = _batch(new, total, d, dtype, block, 5)
    out, lse = _call(q, starts, k, ks, v, vs, table, total, 0.1)
    for r, n in enumerate(new):
        if n == 0:
            continue
        a, b = starts[r], starts[r + 1]
        blind = max(0, n - total[r])
        assert bool((out[a:a + blind] == 0).all()) and bool((lse[a:a + blind] == -math.inf).all())
        kk, vv = R.gather(k, ks, table[r], total[r], block), R.gather(v, vs, table[r], total[r], block)
        _close(out[a:b], lse[a:b], q[a:b], kk, vv, _key_scales(vs, table[r], total[r], block), [total[r] - n + 1 + i for i in range(n)], 0.1, 4,
               chunk=True)
    for cu in ([0, 100, 200, 300], [-5, 6, 12, 41], [8, 3, 12, 0], [41, 41, 41, 41], [2 ** 31 - 1, -2 ** 31, 0, 7]):
        _call(q, cu, k, ks, v, vs, table, total, 0.1)
    _call(q, starts, k, ks, v, vs, table, [2 ** 31 - 1, -3, 40], 0.1)
    torch.cuda.synchronize()


@pytest.mark.parametrize("h,hk,d,dtype", [(40, 2, 256, torch.bfloat16), (34, 1, 256, torch.float16), (48, 1, 128, torch.bfloat16), (140, 1, 128, torch.float16)])
def test_decode_of_wide_groups(h, hk, d, dtype):
    assert _chunk(dtype, d, 1, h // hk, 1)
    _decode_case([1, 0, 15, 16, 17, 127, 128, 129, 0, 255, 64, 700], h, hk, d, 32, dtype, seed=h)


@pytest.mark.parametrize("new,d,dtype", _MANY)
def test_nan_and_infinite_operands_reach_their_rows_only(new, d, dtype):
    """A NaN key reaches the tokens that see it, a NaN or infinite query its own row."""
    total, block = [200, 150, 90], 16
    k, ks, v, vs, table, starts, q = _batch(new, total, d, dtype, block, 9)
    held = total[0] - new[0]
    at = held + new[0] // 2                                          # a key of the call's own
    k.view(torch.uint8)[table[0, at // block], 0, at % block, 5] = 0x7F
    last = starts[-1] - 1
    q[last, 2], q[last, 3, 7] = math.inf, math.nan
    out, lse = (x.cpu() for x in _call(q, starts, k, ks, v, vs, table, total, 0.1))
    sees = torch.zeros(starts[-1], 8, dtype=torch.bool)
    sees[at - held:new[0], :4] = True
    sees[last, 2:4] = True
    assert torch.equal(torch.isnan(out).any(2), sees) and torch.equal(torch.isnan(out).all(2), sees)
    assert torch.equal(torch.isnan(lse), sees)


@pytest.mark.parametrize("d", [128, 256])
def test_a_chunk_by_itself_and_among_idle_rows(d):
    """The rows of the table that a chunk needs, or all of it: other kernels, the same attention."""
    rows, n, total, block = 40, 60, [0] * 17 + [300] + [0] * 22, 16
    k, ks = _cache(25, 2, block, d, 3)
    v, vs = _cache(25, 2, block, d, 53)
    table = _table(total, block, 25, 1)
    _spoil(k, ks, table, total, block)
    _spoil(v, vs, table, total, block)
    q = torch.randn(n, 8, d, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    kk, vv = R.gather(k, ks, table[17], 300, block), R.gather(v, vs, table[17], 300, block)
    cu = [0] * 18 + [n] * 23
    for a, b, chunk in ((0, rows, False), (17, 18, True)):
        assert _chunk(torch.bfloat16, d, n, 4, b - a) == chunk
        whole, lengths = table.cuda(), _i32(total)
        out, lse = _nv().fp8_paged_attention(q.cuda(), _i32(cu[a:b + 1]), k.cuda(), v.cuda(), ks.cuda(), vs.cuda(), whole[a:b], lengths[a:b], 0.1, 4,
                                             return_lse=True)
        _close(out, lse, q, kk, vv, _key_scales(vs, table[17], 300, block), [241 + i for i in range(n)], 0.1, 4, chunk=chunk)


@pytest.mark.parametrize("new,d,dtype", [([3, 1, 2], 128, torch.bfloat16), ([2, 3, 1], 256, torch.float32), _MANY[0], _MANY[3]])
def test_blocks_whose_offsets_pass_32_bits(new, d, dtype):
    """A view of a wider buffer, half a gigabyte from block to block: written and read through both kernels."""
    hk, block, apart = 2, 64, (1 << 29) + 4096
    total = [130, 61, 90]
    blocks = sum(-(-n // block) for n in total) + 4                  # 4.5 GB and more
    assert (blocks - 1) * apart > 1 << 32
    flat = torch.empty(blocks * apart, dtype=torch.uint8, device="cuda")
    view = lambda at: flat.as_strided((blocks, hk, block, d), (apart, block * d, d, 1), at)
    k, v = view(0), view(1 << 20)
    k.zero_(), v.zero_()
    ks, vs = torch.zeros(blocks, hk, device="cuda"), torch.zeros(blocks, hk, device="cuda")
    table = _table(total, block, blocks, 2)
    g = torch.Generator().manual_seed(4)
    assert int(table.max()) * apart > 1 << 32
    slots = [int(table[r, p // block]) * block + p % block for r, n in enumerate(total) for p in range(n)]
    key, value = (torch.randn(len(slots), hk, d, generator=g) for _ in range(2))
    _nv().fp8_kv_write(key.cuda(), value.cuda(), torch.tensor(slots).cuda(), k, v, ks, vs)
    wk, wv = torch.zeros(blocks, hk, block, d).double(), torch.zeros(blocks, hk, block, d).double()
    wks, wvs = torch.zeros(blocks, hk).double(), torch.zeros(blocks, hk).double()
    R.write(key.double(), slots, wk, wks, block)
    R.write(value.double(), slots, wv, wvs, block)
    for got, s, want, ws in ((k, ks, wk, wks), (v, vs, wv, wvs)):
        assert torch.equal(s.cpu().double(), ws)
        assert torch.equal(got.cpu().view(torch.float8_e4m3fn).double(), want)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = torch.randn(starts[-1], 4 * hk, d, generator=g).to(dtype)
    out, lse = _nv().fp8_paged_attention(q.cuda(), _i32(starts), k, v, ks, vs, table.cuda(), _i32(total), 0.1, 4, return_lse=True)
    for r, n in enumerate(new):
        if n:
            a, b = starts[r], starts[r + 1]
            kk, vv = R.gather(wk, wks, table[r], total[r], block), R.gather(wv, wvs, table[r], total[r], block)
            _close(out[a:b], lse[a:b], q[a:b], kk, vv, _key_scales(wvs, table[r], total[r], block), [total[r] - n + 1 + i for i in range(n)], 0.1, 4,
                   chunk=_chunk(dtype, d, starts[-1], 4, 3))
